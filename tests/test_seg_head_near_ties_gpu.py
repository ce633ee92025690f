"""Alternatives from features where logits are a few units in the last place apart, or equal: the order of classes.

Every product is 0 or 1 and the bias a small multiple of one unit: the fp32 sum of both is exact, so the reference's logits are the operator's and
its classes have to be equal."""
import pytest
import torch

from test_seg_head_scores_gpu import check

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -23          # of numbers from 1 to 2


def head_of(units, base=None, sign=1.0):
    """Features of 16 kinds of rows and weights whose logits are sign * base[kind, class] + sign * units[class] * ULP."""
    K = len(units)
    feat = torch.eye(16, device="cuda").repeat(9, 1)[:140].bfloat16()
    weight = (torch.ones(K, 16) if base is None else base.t().float()).cuda()
    return feat, (sign * weight).bfloat16(), (sign * torch.as_tensor(units).double() * ULP).cuda().bfloat16()


@pytest.mark.parametrize("top", [1, 2, 7, 8, 15, 16, 17, 32])
@pytest.mark.parametrize("K", [32, 64, 100, 1201])
def test_one_logit_larger_than_equal_ones(K, top):
    """At every place of 32, one to 31 units above all others: alone, and behind as many larger ones as leave it the last place or the one behind."""
    for place in list(range(32)) + [K - 1]:
        units = torch.zeros(K)
        units[place] = (1, 8, 31)[place % 3]
        check(*head_of(units), None, top)
    for larger in {top - 2, top - 1, top} & set(range(1, 31)):
        units = torch.zeros(K)
        units[:larger] = 64                     # (beyond the 32 units that may look alike)
        units[31] = 1
        check(*head_of(units), None, top)


@pytest.mark.parametrize("sign", [1.0, -1.0], ids=["above", "below"])
@pytest.mark.parametrize("K", [20, 32, 33, 64, 130, 700])
def test_logits_of_few_units(K, sign):
    """Logits of 2, 5, 32 and 200 different values within as many units, where each row has another half of the classes."""
    g = torch.Generator().manual_seed(K)
    for values in (2, 5, 32, 200):
        units = torch.randint(0, values, (K,), generator=g)
        base = (torch.rand(16, K, generator=g) < 0.5).float()
        base[0], base[1] = 1, 0                 # all of them, none (logits of a few 2^-23)
        for top in (1, 3, 8, 16, 31):
            check(*head_of(units, base, sign), None, top)


@pytest.mark.parametrize("K", [40, 300])
def test_rising_and_falling_units(K):
    for units in (torch.arange(K) % 32, 31 - torch.arange(K) % 32, torch.arange(K) // 8 % 32):
        for top in (1, 8, 16, 32):
            check(*head_of(units), None, top)
