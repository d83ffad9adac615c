"""The embedding's gradient at the ends of its ranges. Values are small whole numbers, so that sums in f32 are exact: every row has to be equal."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def test_as_many_classes_as_there_can_be():
    """2^31 - 1 classes of one feature, of few positions: the last ones are written as the first, and no row is left as it was."""
    from mimir_b200 import _lib
    from mimir_b200 import tensor as T
    v = 2 ** 31 - 1
    for id_dtype, code in ((torch.int32, _lib.I32), (torch.int64, _lib.I64)):
        ids = torch.tensor([0, v - 1, 1, v - 2, 1 << 30, v - 1, v - 1024, 1023], dtype=id_dtype, device="cuda")
        dy = torch.arange(1, 9, device="cuda", dtype=F32).to(BF16).view(8, 1)
        out = torch.full((v, 1), float("nan"), dtype=BF16, device="cuda")
        d = _lib.EmbeddingDesc()
        d.n, d.d, d.v, d.ids, d.dy, d.dtable, d.scale = 8, 1, v, ids.data_ptr(), dy.data_ptr(), out.data_ptr(), 1.0
        d.dtype, d.out_dtype, d.id_dtype = _lib.BF16, _lib.BF16, code
        assert _lib.lib().mimk_embedding_grad(C.byref(d), torch.cuda.current_stream().cuda_stream) == 0
        there = {0: 1, 1: 3, 1023: 8, 1 << 30: 5, v - 1024: 7, v - 2: 4, v - 1: 2 + 6}
        assert all(float(out[c]) == w for c, w in there.items())
        for c in there:
            out[c] = 0
        assert not any(bool(part.ne(0).any()) for part in out.split(1 << 28))
        del out
    T.device_status()
