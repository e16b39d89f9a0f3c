"""Every launch stands inside its tensors' device, whichever is the current one: where one GPU is all there is, by watching when the
stream is asked for."""

import contextlib

import pytest

pytestmark = pytest.mark.gpu


def test_launches_are_made_on_the_tensors_device(monkeypatch):
    import torch
    from nkilib import _native as nv
    from nkilib.core.cumsum import cumsum
    from nkilib.core.moe.glu_checkpoint import dequantize_checkpoint, glu_checkpoint, glu_checkpoint_bwd, pack_gate_up_checkpoint
    from nkilib.core.moe.moe_cte import build_token_blocks
    from nkilib.core.moe.token_permute import build_token_slots, combine_tokens, combine_tokens_bwd, permute_tokens, permute_tokens_bwd
    from nkilib.core.router_topk import route_for_moe, router_topk, router_topk_bwd
    from nkilib.core.subkernels import find_nonzero_indices, indexed_flatten
    from nkilib.core.utils.common_types import RouterActFnType

    inside, asked = [], []
    real = nv.stream_ptr

    @contextlib.contextmanager
    def on_device(device):
        inside.append(device)
        yield
        inside.pop()

    def stream_ptr(device):
        asked.append(inside[-1:] == [device])
        return real(device)

    monkeypatch.setattr(nv, "on_device", on_device)
    monkeypatch.setattr(nv, "stream_ptr", stream_ptr)
    T, H, E, k, B = 24, 128, 8, 2, 4
    r = lambda *s: torch.randn(s, device="cuda").bfloat16()
    x, w = r(T + 1, H), r(H, E)
    state = {}

    def route():
        state["ids"], state["aff"], state["logits"] = route_for_moe(x, w, None, k, RouterActFnType.SOFTMAX, True, return_router_logits=True)

    def blocks():
        state["tp"], state["be"], _ = build_token_blocks(state["ids"], E, B)

    def sums():
        a = (state["aff"], state["tp"], state["be"], B)
        xs = permute_tokens(x[:T], state["tp"])
        combine_tokens(xs, *a, T, k)
        combine_tokens_bwd(x[:T], xs, *a, k)
        permute_tokens_bwd(xs, state["tp"], T, k)
        build_token_slots(state["tp"], T, k)

    def glu():
        h, c, s = glu_checkpoint(r(6, 2, 32))
        glu_checkpoint_bwd(c, s, h)
        dequantize_checkpoint(c, s)
        pack_gate_up_checkpoint(r(2, 2, 32, 4))

    calls = {
        "router_topk": lambda: router_topk(x, w, None, None, None, None, RouterActFnType.SOFTMAX, k, x_hbm_layout=1),
        "route_for_moe": route,
        "build_token_blocks": blocks,
        "rows": sums,
        "glu": glu,
        "router_topk_bwd": lambda: router_topk_bwd(state["aff"], x[:T], w, None, state["logits"], state["ids"], RouterActFnType.SOFTMAX,
                                                   norm_topk_prob=True),
        "cumsum": lambda: cumsum(torch.ones((3, 8), device="cuda")),
        "find_nonzero_indices": lambda: find_nonzero_indices(torch.ones((8, 3), dtype=torch.int32, device="cuda")),
        "indexed_flatten": lambda: indexed_flatten(torch.ones((2, 8), dtype=torch.int32, device="cuda"), 4, 16,
                                                   torch.zeros(2, dtype=torch.int32, device="cuda")),
    }
    for name, call in calls.items():
        asked.clear()
        call()
        assert asked and all(asked), name
