"""CPU test of where the launches of the layer on 4-bit experts go: all of them to the tensors' own device, whichever
is current.  The launches are recorded instead of made."""
import pytest
import torch

E, H, I, T, K = 32, 64, 8, 3, 2


@pytest.mark.parametrize("fused", [False, True])
def test_every_launch_is_on_the_tensors_device(monkeypatch, fused):
    from sonicmoe import functional as fn

    seen = []
    monkeypatch.setattr(fn.ops, "_need", lambda *a: None)
    monkeypatch.setattr(fn.ops, "_call_on", lambda device, name, *a: seen.append((device.type, name)))
    monkeypatch.setattr(fn.ops.nat, "call", lambda *a: pytest.fail(f"{a[0]} goes to the current device"))
    monkeypatch.setattr(fn.ops, "_workspace", lambda n, device: torch.empty(16, dtype=torch.uint8, device=device))
    w = [fn.ops.Int4ExpertWeights(torch.empty(1024 * b), torch.empty(64 * b), shape, 32, False)
         for b, shape in ((E, (E, 2 * I, H)), (4 * E, (E, H, I)))]
    x = torch.zeros(T, H, dtype=torch.bfloat16)
    fn.moe_TC_softmax_topk_layer(x, torch.zeros(E, H), w[0], None, w[1], None, K, None, is_inference_mode_enabled=True,
                                 fused_router=fused)
    assert seen == [("cpu", "sm_router_fused" if fused else "sm_router_topk"), ("cpu", "sm_moe_int4_forward")]
