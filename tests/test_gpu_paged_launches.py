"""What the paged cache's calls launch."""
import json

import pytest
import torch

from _paged import Cache, ptr

pytestmark = pytest.mark.gpu


def kernels(tmp_path, call):
    """(name, arguments) of the kernels that call launches, from the profiler's trace."""
    call()
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        call()
        torch.cuda.synchronize()
    path = tmp_path / "trace.json"
    prof.export_chrome_trace(str(path))
    found = [(e["name"], e["args"]) for e in json.loads(path.read_text())["traceEvents"] if e.get("cat") == "kernel"]
    if not found:
        pytest.skip("the profiler sees no kernels (another one may be at work)")
    return found


@pytest.mark.parametrize("kind,D", [("f16", 32), ("bf16", 32), ("f16", 64), ("bf16", 64), ("f32", 32), ("bf16", 128), ("f32", 256)])
def test_the_weights_blocks_are_resident_at_once(cuda_engine, torch_cuda, tmp_path, kind, D):
    """Their work is split evenly: a block that waits for another to end would run its share alone."""
    cache = Cache(kind, 4, D, 16, [300, 200])
    q, out = torch.randn(2, 8, D, device="cuda"), torch.zeros(2, 8, D, device="cuda")
    lse, weights = torch.zeros(2, 8, device="cuda"), torch.zeros(2, 4, cache.cap, device="cuda")
    lens = torch.tensor([300, 200], dtype=torch.int32, device="cuda")
    found = kernels(tmp_path, lambda: cache.handle(cuda_engine).attention(
        ptr(q), 8, 2, ptr(lens), ptr(out), lse_ptr=ptr(lse), weights_ptr=ptr(weights)))
    args = [a for name, a in found if "paged_weights" in name]
    assert len(found) == 2 and len(args) == 1, [n for n, _ in found]
    blocks, threads = args[0]["grid"][0], args[0]["block"][0]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    registers = 32 * -(-args[0]["registers per thread"] // 8) * 8  # of a warp, in steps of 256
    fit = min(65536 // (registers * threads // 32), 228 * 1024 // (args[0]["shared memory"] + 1024))
    assert blocks % sms == 0 and 1 <= blocks // sms <= fit, (blocks, sms, fit, args[0])
