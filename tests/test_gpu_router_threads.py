"""GPU test of the fused router called from several host threads at once with other numbers of experts, which
take the same kernel with different amounts of shared memory."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_threads():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from sonicmoe import _native as nat
    from sonicmoe import ops

    T, H, K = 256, 256, 4
    lib, jobs, keep = nat.load(), [], []
    for E in (32, 128, 32, 128):
        g = torch.Generator(device="cuda").manual_seed(E)
        x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
        w = torch.randn(E, H, generator=g, device="cuda").to(torch.bfloat16)
        want, _, _ = ops.router_fused(x, w, K)
        logits, scores, idx = (torch.empty_like(want), torch.empty(T, K, device="cuda"),
                               torch.empty(T, K, dtype=torch.int32, device="cuda"))
        ws = torch.empty(lib.sm_router_fused_workspace(T, E), dtype=torch.uint8, device="cuda")
        err, stream = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.cuda.Stream()
        jobs.append(((x.data_ptr(), w.data_ptr(), T, H, E, K, 1, 0, logits.data_ptr(), scores.data_ptr(), idx.data_ptr(),
                      ws.data_ptr(), ws.numel(), err.data_ptr(), stream.cuda_stream), stream, logits, want))
        keep.append((x, w, scores, idx, ws, err))
    torch.cuda.synchronize()
    start, failed = threading.Barrier(len(jobs)), []

    def work(args, stream, out, want):
        torch.zeros(1, device="cuda")  # a context is current in this thread
        start.wait()
        for _ in range(4000):
            if lib.sm_router_fused(*args):
                failed.append(lib.sm_last_error().decode())
                break
        stream.synchronize()
        if not torch.equal(out, want):
            failed.append("another result")

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
