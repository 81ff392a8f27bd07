"""GPU tests of the 4-bit experts called from several host threads at once, each with its own stream, and sizes
that take the same kernels with different amounts of shared memory."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first,second", [((1, 8), (8, 8)), ((3, 4), (3, 3000)), ((40, 4), (40, 1000)),
                                          ((200, 6), (600, 10))])
def test_threads(first, second):
    """(tokens, experts) of two threads each; every call gives what it gives alone."""
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from sonicmoe import ops

    from sonicmoe import _native as nat

    H, I, K = 256, 128, 4
    lib, jobs, keep = nat.load(), [], []
    for i, (T, E) in enumerate((first, second)):
        g = torch.Generator(device="cuda").manual_seed(i)
        w1 = torch.randn(E, 2 * I, H, generator=g, device="cuda", dtype=torch.bfloat16) * 0.02
        w2 = torch.randn(E, H, I, generator=g, device="cuda", dtype=torch.bfloat16) * 0.02
        x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
        idx = torch.rand(T, E, generator=g, device="cuda").topk(K, 1).indices.to(torch.int32)
        scores = torch.rand(T, K, generator=g, device="cuda")
        p1, p2 = ops.weight_prep_int4(w1, 64), ops.weight_prep_int4(w2, 64)
        want, _ = ops.moe_int4_forward(x, scores, idx, p1, p2)
        for _ in range(2):  # the entry point itself, so that the calls follow each other closely
            out = torch.empty_like(x)
            freq = torch.empty(E, dtype=torch.int32, device="cuda")
            ws = torch.empty(lib.sm_moe_int4_workspace_bytes(T, T * K, H, I, E), dtype=torch.uint8, device="cuda")
            stream = torch.cuda.Stream()
            ptr = [t.data_ptr() for t in (x, scores, idx, p1.q, p1.scales, p2.q, p2.scales, out, freq, ws)]
            args = (ptr[0], T, H, I, E, K, T * K, ptr[1], None, ptr[2], ptr[3], ptr[4], 64, ptr[5], ptr[6], 64, ptr[7],
                    ptr[8], ptr[9], ws.numel(), None, stream.cuda_stream)
            jobs.append((args, stream, out, want))
            keep.append((x, scores, idx, p1, p2, freq, ws))
    torch.cuda.synchronize()
    start, failed = threading.Barrier(len(jobs)), []

    def work(args, stream, out, want):
        start.wait()
        for _ in range(4000):
            if lib.sm_moe_int4_forward(*args):
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
