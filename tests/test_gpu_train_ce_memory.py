"""The F32 cross-entropy of a linear layer plans all its memory: no call allocates on the device, and one that is captured runs the kernels of one that is
not, to the same bits. Sizes at which the library's f32 products cut their operands beforehand, into scratch."""
import ctypes as C

import pytest
import torch

from test_gpu_train_ce import F32, IGNORED, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(2048, 512, 8192), (2049, 516, 8196), (1500, 128, 131072), (512, 784, 10007)])
@pytest.mark.parametrize("masked", [0.0, 0.3])
@pytest.mark.parametrize("nk", [False, True])
def test_same_bits_in_a_graph(shape, masked, nk):
    from mimir_b200 import tensor as T
    x, w, t = inputs(*shape, F32, nk, masked=masked)
    ignore = IGNORED if masked else None

    def calls():
        losses, lse = T.linear_cross_entropy(x, w, t, ignore_index=ignore, reduction="none", return_lse=True)
        return (losses, lse) + T.linear_cross_entropy_with_grad(x, w, t, ignore_index=ignore) + T.linear_cross_entropy_grad(x, w, t, lse, ignore_index=ignore)

    want = calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for g in got:
        g.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    T.device_status()


def test_no_allocation():
    """(One would do for a cached buffer that had to grow: the second size is beyond what the first and other tests leave behind. The first loads the kernels.)"""
    from mimir_b200 import _lib
    L = _lib.lib()
    for n, d, v in ((2048, 512, 8192), (6000, 4000, 20000)):
        x, w, t = inputs(n, d, v, F32, True)
        loss, lse, dx, dw = (torch.empty(s, device="cuda") for s in ((), (n,), (n, d), (v, d)))
        desc, need = _lib.LinearCeDesc(), C.c_uint64()
        desc.n, desc.d, desc.v, desc.dtype, desc.target_dtype, desc.w_layout, desc.reduction = n, d, v, _lib.F32, _lib.I64, _lib.B_NK, _lib.REDUCTION_MEAN
        desc.x, desc.w, desc.targets, desc.loss, desc.lse, desc.dx, desc.dw = (a.data_ptr() for a in (x, w, t, loss, lse, dx, dw))
        room = 0
        for forward, backward in ((1, 0), (1, 1), (0, 1)):
            assert L.mimk_linear_ce_workspace(C.byref(desc), forward, backward, C.byref(need)) == 0
            room = max(room, need.value)
        ws = torch.empty(room, dtype=torch.uint8, device="cuda")
        desc.workspace, desc.workspace_bytes = ws.data_ptr(), room
        stream = torch.cuda.current_stream().cuda_stream
        torch.cuda.synchronize()
        free = torch.cuda.mem_get_info()[0]
        for call in (L.mimk_linear_ce_fwd, L.mimk_linear_ce_fwd_bwd, L.mimk_linear_ce_bwd):
            assert call(C.byref(desc), stream) == 0
        torch.cuda.synchronize()
    assert torch.cuda.mem_get_info()[0] == free
