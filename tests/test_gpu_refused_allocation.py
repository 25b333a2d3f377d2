"""A call that the device's memory does not suffice for is refused, and nothing else notices."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TOO_MANY = 1 << 30  # pages of one slot: terabytes


def test_the_next_calls_go_on(cuda_engine, tools, torch_cuda):
    img = tools.synth_gguf(tools.TINY)
    eng = cuda_engine.Engine(img, 64)
    b = cuda_engine.Batch(eng, 2, 64)
    refs = cuda_engine.Batch(eng, 2, 64)
    rows = [b.forward([0], [1])[0]]
    want = [refs.forward([0], [1])[0]]
    for t in (2, 3):
        with pytest.raises(cuda_engine.QwenCudaError, match="out of memory") as ei:
            cuda_engine.Batch.paged(eng, 1, 64, cuda_engine.PagedCache.F32, 1, TOO_MANY)
        assert ei.value.code == cuda_engine.ERR_NOMEM
        rows.append(b.forward([0], [t])[0])
        want.append(refs.forward([0], [t])[0])
    assert b.position(0) == 3
    assert all(np.array_equal(r, w) for r, w in zip(rows, want))
    # the same before calls on arrays of one's own
    with pytest.raises(cuda_engine.QwenCudaError, match="out of memory"):
        cuda_engine.Batch.paged(eng, 1, 64, cuda_engine.PagedCache.F32, 1, TOO_MANY)
    k = torch_cuda.ones(2, 1, 16, 64, device="cuda")
    v = torch_cuda.ones_like(k)
    table = torch_cuda.zeros(1, 1, dtype=torch_cuda.int32, device="cuda")
    pos = torch_cuda.full((1,), 3, dtype=torch_cuda.int32, device="cuda")
    row = torch_cuda.full((1, 1, 64), 5.0, device="cuda")
    cache = cuda_engine.PagedCache(cuda_engine.PagedCache.F32, k.data_ptr(), v.data_ptr(), 2, 16, 1, 64, table.data_ptr(), 1, 1)
    cache.append(row.data_ptr(), row.data_ptr(), 1, pos.data_ptr())
    torch_cuda.cuda.synchronize()
    assert bool((k[0, 0, 3] == 5).all()) and int((k == 5).sum()) == 64
