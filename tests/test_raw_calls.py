"""Calls that functional.py has checked forms of: tensors that the kernels cannot read are refused all the same, before a launch."""
import pytest
import torch

from pointtransformerv3_b200 import _lib, ops

X, LIST = torch.zeros(4, 5), torch.zeros(4, 2, dtype=torch.int32)
STATUS = torch.zeros(1, dtype=torch.int32)


@pytest.mark.parametrize("grad", [False, True])
def test_tensors_of_the_host_are_refused(grad):
    x = X.clone().requires_grad_(grad)
    before = _lib.load().ptv3_launch_count()
    for call in (lambda: ops.class_scores(x, None, 2, 1.0, -1, None),
                 lambda: ops.class_scores(x, torch.zeros(4, dtype=torch.int64), 0, 1.0, -1, STATUS),
                 lambda: ops.distill_topk(x, torch.zeros(4, 2), LIST, 1.0, False, STATUS)):
        with pytest.raises(_lib.Ptv3Error, match="CUDA kernels only"):
            call()
    assert _lib.load().ptv3_launch_count() == before


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
def test_types_that_the_kernels_do_not_have_are_refused(dtype):
    x, status = X.cuda(), ops.new_status("cuda")
    values = torch.zeros(4, 2, device="cuda")
    for call in (lambda: ops.class_scores(x.to(dtype), None, 2, 1.0, -1, None),
                 lambda: ops.distill_topk(x.to(dtype), values, LIST.cuda(), 1.0, False, status),
                 lambda: ops.distill_topk(x, values.to(dtype), LIST.cuda(), 1.0, False, status)):
        with pytest.raises(_lib.Ptv3Error, match="dtype"):
            call()


@pytest.mark.gpu
def test_a_tensor_of_the_host_among_others_is_refused():
    x, status = X.cuda(), ops.new_status("cuda")
    for call in (lambda: ops.class_scores(x, torch.zeros(4, dtype=torch.int64), 0, 1.0, -1, status),
                 lambda: ops.class_scores(x, torch.zeros(4, dtype=torch.int64).cuda(), 0, 1.0, -1, STATUS),
                 lambda: ops.distill_topk(x, torch.zeros(4, 2), LIST.cuda(), 1.0, False, status),
                 lambda: ops.distill_topk(x, torch.zeros(4, 2).cuda(), LIST, 1.0, False, status),
                 lambda: ops.distill_topk(x, torch.zeros(4, 2).cuda(), LIST.cuda(), 1.0, False, STATUS)):
        with pytest.raises(_lib.Ptv3Error, match="CUDA kernels only"):
            call()
