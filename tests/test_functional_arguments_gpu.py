"""Arguments of the trainable operators as programs have them: slices of larger buffers, tensors that change, other modes of torch."""
import pytest
import torch

import functional_reference as R
from pointtransformerv3_b200 import functional as F

pytestmark = pytest.mark.gpu


def normal(*shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [8, 16, 64, 128])
def test_weights_from_a_buffer_of_parameters(D, dtype):
    """Norm weights that are slices of one buffer, behind an odd number of values: the same bits as copies of them, forward and
    in all gradients."""
    n, heads = 77, 2
    qkv = normal(n, 3 * heads * D, seed=1, dtype=dtype)
    dout = normal(n, 3 * heads * D, seed=2, dtype=dtype)
    buffer = 1 + normal(2 * D + 9, seed=3, dtype=dtype, scale=0.2)
    grid = torch.randint(0, 99, (n, 3), generator=torch.Generator().manual_seed(4), dtype=torch.int32).cuda()

    def run(q, k):
        x, q, k = (t.detach().requires_grad_() for t in (qkv, q, k))
        out = F.qk_norm_rope(x, heads, grid, q, k)
        return (out,) + torch.autograd.grad(out, (x, q, k), dout)
    for first in (0, 1, 2, 3, 5):
        q, k = buffer[first:first + D], buffer[first + D + 1:first + 2 * D + 1]
        assert (q.data_ptr() - buffer.data_ptr()) == first * buffer.element_size()
        assert all(torch.equal(a, b) for a, b in zip(run(q, k), run(q.clone(), k.clone())))
