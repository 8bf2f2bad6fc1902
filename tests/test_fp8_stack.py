"""The decoder stack with its projections in e4m3: every call of a pass against
64-bit arithmetic on what that call was given and on the weights as the model
holds them, and each call's result as the next one's input.  (A pass from end
to end has no bound worth testing: a value next to the border of two e4m3
values goes to the other one for the smallest reason.)"""
import numpy as np
import pytest
import torch

import cev_hip
from cev_hip import Fp8Rows, configs
from test_fp8 import E4M3, E8M0, check_gate_up, check_product, check_rows_near, oracle_blocks, oracle_norm, oracle_rows, values, weight_of, weight_values


def tiny(bf16, **kw):
    sizes = dict(n_layers=2, hidden=256, hq=4, hkv=2, d=128, inter=648, vocab=512, state_tokens=96, prefill_chunk=64, questions=3, q_len=5)
    return configs.Qwen3StackWorkload("tiny", 9, bf16, **{**sizes, **kw})


def e4m3_of(x):
    """(values, scales) of a float weight, on the CPU."""
    q, e = oracle_blocks(x)
    return q.float().to(E4M3), (e + 127).to(torch.uint8).view(E8M0)


def weights_of(w, kind):
    """The stack's weights, and each projection's values in 64 bits: floats (quantised by the stack) or a checkpoint's pairs."""
    weights = w.weights()
    true = {}
    for name, _, (n, k) in w.weight_specs():
        if name == "embed":
            continue
        if kind == "floats":
            true[name] = torch.from_numpy(weights[name])
        else:
            weights[name] = weight_of(n, k, kind, len(true) + 50)
            true[name] = weight_values(*weights[name]) * 2.0 ** -4
            weights[name] = (weights[name][0], (weights[name][1].float() * 2.0 ** -4).to(weights[name][1].dtype))
    layers = []
    for i in range(w.n_layers):
        p = f"l{i}."
        one = {"wqkv": torch.cat([true[p + x] for x in ("wq", "wk", "wv")]), "wo": true[p + "wo"], "gate": true[p + "gate"], "up": true[p + "up"],
               "wdown": true[p + "down"]}
        layers.append({n: weight_values(*e4m3_of(x)) if kind == "floats" else x for n, x in one.items()})
    return weights, layers


def copied(x):
    return Fp8Rows(x.q.clone(), x.s.clone(), x.k) if isinstance(x, Fp8Rows) else x.clone() if isinstance(x, torch.Tensor) else x


def same(a, b):
    if isinstance(a, Fp8Rows):
        return isinstance(b, Fp8Rows) and torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.s.view(torch.uint8), b.s.view(torch.uint8))
    return torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kind", ["floats", "e8m0", "f32"])
def test_every_call_of_a_pass(gpu, monkeypatch, kind, bf16):
    from cev_hip import qwen3
    w = tiny(bf16)
    weights, layers = weights_of(w, kind)
    stack = qwen3.Qwen3Stack(w, weights, gpu, capacity=160, fp8=True)
    calls = []
    for name in ("rms_norm_fp8", "linear_fp8", "gate_up_fp8"):
        def recorded(x, *a, _name=name, _f=getattr(qwen3, name), **kw):
            given = [copied(y) for y in (x, kw.get("h"))]
            r = _f(x, *a, **kw)
            calls.append((_name, given, copied(r), copied(x)))
            return r
        monkeypatch.setattr(qwen3, name, recorded)
    tab, pos, slots, gather = cev_hip.BlockTable.from_slots([(0, 70, 0)], [], 160)
    x, h = stack.run(np.arange(70) * 7 % w.vocab, pos, slots, tab)
    assert [c[0] for c in calls] == ["rms_norm_fp8", "linear_fp8", "linear_fp8", "rms_norm_fp8", "gate_up_fp8", "linear_fp8"] * w.n_layers
    dtype = torch.bfloat16 if bf16 else torch.float32

    def norm(call, k=w.hidden):
        _, (before, res), rows, after = call
        xo, want = oracle_norm(before.cpu(), torch.ones(k), w.eps, None if res is None else res.cpu(), False)
        assert torch.equal(after.double().cpu(), xo)
        check_rows_near(rows, want, (k / 128 + 24) * 2.0 ** -24)  # as for the norm itself

    def operand(x):
        if isinstance(x, Fp8Rows):
            return values(x.q.cpu(), x.s.cpu())[:, : x.k]
        q, e = oracle_rows(x.cpu())
        return (q * torch.exp2(e).repeat_interleave(128, 1))[:, : x.shape[1]]

    for i, L in enumerate(layers):
        ln1, qkv, wo, ln2, gu, down = calls[6 * i: 6 * i + 6]
        norm(ln1)
        assert same(ln1[2], qkv[1][0])
        check_product(qkv[2], operand(qkv[1][0]), L["wqkv"], dtype)
        check_product(wo[2], operand(wo[1][0]), L["wo"], dtype)
        assert same(wo[2], ln2[1][1]) and same(ln1[3], ln2[1][0])
        norm(ln2)
        assert same(ln2[2], gu[1][0])
        check_gate_up(gu[2], operand(gu[1][0]), L["gate"], L["up"])
        assert same(gu[2], down[1][0])
        check_product(down[2], operand(down[1][0]), L["wdown"], dtype)
        if i + 1 < len(layers):
            nxt = calls[6 * i + 6]
            assert same(down[2], nxt[1][1]) and same(ln2[3], nxt[1][0])
    assert same(h, calls[-1][2]) and same(x, calls[-3][3])


@pytest.mark.gpu
def test_engine_over_an_e4m3_stack(gpu):
    """The engine's whole flow, twice: a prefix that is cached the second time."""
    from cev_hip.engine import DeviceEngine
    from cev_hip.qwen3 import Qwen3Stack
    w = tiny(True)
    state, qs, codes = w.ids()
    stack = Qwen3Stack(w, w.weights(), gpu, capacity=256, fp8=True)
    eng = DeviceEngine(stack, budget=w.state_tokens, code_ids=codes, pass_tokens=w.pass_tokens, prefill_chunk=w.prefill_chunk)
    first, second = (eng.run_many([(state, list(qs))])[0] for _ in range(2))
    assert not first["prefix_cached"] and second["prefix_cached"]
    for r in (first, second):
        assert r["logits"].shape == (w.questions, w.n_codes) and np.isfinite(r["logits"]).all()


@pytest.mark.gpu
def test_joined_weights_want_whole_blocks(gpu):
    from cev_hip.qwen3 import Qwen3Stack
    w = tiny(True, hq=1, hkv=1, d=64)
    weights, _ = weights_of(w, "e8m0")
    with pytest.raises(ValueError, match="whole blocks"):
        Qwen3Stack(w, weights, gpu, capacity=64, fp8=True)
    weights, _ = weights_of(tiny(True), "e8m0")
    weights["l0.wk"] = torch.zeros(256, 256)
    with pytest.raises(ValueError, match="together"):
        Qwen3Stack(tiny(True), weights, gpu, capacity=64, fp8=True)
