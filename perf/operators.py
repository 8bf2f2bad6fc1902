"""The calls of a serving step over a paged K/V cache whose time counts.

Four kinds of case:

  tables  the step's bookkeeping from the requests' lengths: pages taken from
          and given back to the free ring, block tables, row offsets,
          positions and cache slots (cev_hip.paged_tables);
  rope    rotary positions of q and k, with the rows of k and v stored in
          their slots of the paged caches, or the gradient's rotation of
          dense rows (cev_hip.rope);
  attend  attention of each request's new tokens over its pages, with or
          without a sliding window and first tokens that stay visible
          (cev_hip.PagedAttention: the work list and the attention);
  step    all of them in a row, as one layer of a serving step runs them.

A host program keeps the caches, the tables' buffers, the rotary angles and
the attention's workspace between calls, so prepare() makes those.  A pass
leaves the state that it started from as it was (the new lengths and the new
ring state go to buffers of their own), so it can be repeated.
"""
import math
import os
import random
import sys

import torch

own = False  # False: run() computes the plain forms; True: the framework's operators

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rust-cev_amd")


def _cev_hip():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import cev_hip
    return cev_hip


# ---------------------------------------------------------------------------
# The cases


def _tables(requests, page, lo, hi, new_lo, new_hi, ended=0.0):
    """requests of lo..hi cached tokens and new_lo..new_hi new ones; a share of `ended` ends instead."""
    return dict(kind="tables", requests=requests, page=page, lo=lo, hi=hi, new_lo=new_lo, new_hi=new_hi, ended=ended)


def _rope(t, hq, hkv, d, bf16, rotary, theta, far, interleaved=False, scaling="none", store=True, page=16):
    """t rows at positions below `far`; store: k and v go to their cache slots, otherwise q and k are gradients of dense rows."""
    return dict(kind="rope", t=t, hq=hq, hkv=hkv, d=d, bf16=bf16, rotary=rotary, theta=theta, far=far, interleaved=interleaved,
                scaling=scaling, store=store, page=page)


def _attend(hq, hkv, d, bf16, page, requests, lo, hi, new_lo, new_hi, window=0, sinks=0, chunked=0):
    """requests of lo..hi cached and new_lo..new_hi new tokens; the first `chunked` of them bring 8 * new_hi instead."""
    return dict(kind="attend", hq=hq, hkv=hkv, d=d, bf16=bf16, page=page, requests=requests, lo=lo, hi=hi, new_lo=new_lo, new_hi=new_hi,
                window=window, sinks=sinks, chunked=chunked)


def _step(hq, hkv, d, bf16, page, requests, lo, hi, new_lo, new_hi, window=0, sinks=0):
    return dict(_attend(hq, hkv, d, bf16, page, requests, lo, hi, new_lo, new_hi, window, sinks), kind="step")


def listed():
    return [
        # a full batch, one token each: the smallest call, all latency
        dict(_tables(64, 16, 100, 4096, 1, 1), name="tables_one_token"),
        # many requests with question-sized chunks, some of them over
        dict(_tables(512, 16, 0, 4096, 17, 64, ended=0.1), name="tables_ragged"),
        # one token of one request on a small model's layer
        dict(_rope(1, 16, 8, 128, True, 128, 1e6, 32768), name="rope_one_token"),
        # a prefill's rows far into a context stretched four times
        dict(_rope(8192, 32, 8, 128, True, 128, 1e6, 131072, scaling="yarn"), name="rope_stretched"),
        # the gradient of a quarter rotary of wide f32 heads, pairs side by side
        dict(_rope(1021, 16, 4, 256, False, 64, 1e7, 8192, interleaved=True, scaling="linear", store=False), name="rope_gradient"),
        # one question's next token on a small model's layer: all latency
        dict(_attend(16, 8, 128, True, 16, 1, 301, 301, 1, 1), name="attend_one_token"),
        # a decoding batch of very different lengths: streaming the K/V cache
        dict(_attend(32, 8, 128, True, 16, 64, 64, 8192, 1, 1), name="attend_decode"),
        # chunks of several prompts over their cached parts
        dict(_attend(32, 8, 128, True, 64, 4, 12000, 32768, 400, 512), name="attend_chunks"),
        # a long prompt's chunk in a layer that sees the last 1024 tokens and the first 4
        dict(_attend(32, 8, 128, True, 32, 2, 1500, 4096, 3500, 4096, window=1024, sinks=4), name="attend_window"),
        # wide heads: a decoding batch with a few question-sized chunks among it
        dict(_attend(16, 4, 256, True, 32, 32, 100, 4096, 1, 8, chunked=4), name="attend_wide_mixed"),
        # an f32 model's question chunks
        dict(_attend(16, 8, 128, False, 16, 12, 256, 2048, 17, 41), name="attend_f32"),
        # a serving step of a small model's layer: bookkeeping, rotary and stores, attention
        dict(_step(16, 8, 128, True, 16, 48, 64, 2048, 1, 4), name="step_small"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "rope", "attend", "attend", "attend", "step"])
    page = rng.choice([16, 16, 32, 64, 128])
    if kind == "tables":
        hi, new_hi = _log(rng, 100, 16384), _log(rng, 1, 64)
        return _tables(_log(rng, 1, 512), page, rng.randint(0, hi), hi, rng.randint(0, new_hi), new_hi, rng.choice([0.0, rng.random() / 2]))
    if kind == "rope":
        hq, hkv, d = rng.choice([(16, 8, 128), (32, 8, 128), (16, 4, 256)])
        return _rope(_log(rng, 1, 8192), hq, hkv, d, rng.random() < 0.7, rng.choice([d, d // 2, d // 4]), rng.choice([1e6, 1e7]),
                     _log(rng, 8192, 1 << 20), rng.random() < 0.4, rng.choice(["none", "linear", "yarn", "wavelength"]), rng.random() < 0.7,
                     page)
    form = rng.choice(["decode", "chunks", "wide", "f32", "window"])
    hq, hkv, d = (16, 4, 256) if form == "wide" else rng.choice([(16, 8, 128), (32, 8, 128)])
    bf16 = form != "f32"
    if kind == "step":
        hi, new_hi = _log(rng, 64, 4096), _log(rng, 1, 16)
        return _step(hq, hkv, d, bf16, page, _log(rng, 1, 64), rng.randint(0, hi), hi, rng.randint(1, new_hi), new_hi)
    if form == "decode":
        hi = _log(rng, 64, 16384)
        return _attend(hq, hkv, d, bf16, page, _log(rng, 1, max(1, min(128, 400000 // hi))), rng.randint(1, hi), hi, 1, rng.choice([1, 1, 3]))
    if form == "window":
        hi, new_hi = _log(rng, 64, 8192), _log(rng, 1, 2048)
        return _attend(hq, hkv, d, bf16, page, _log(rng, 1, max(1, 4096 // new_hi)), rng.randint(1, hi), hi, rng.randint(1, new_hi), new_hi,
                       _log(rng, 32, 2048), rng.choice([0, 1, 4, rng.randint(1, 100)]))
    hi, new_hi = _log(rng, 64, 16384 if form == "chunks" else 4096), _log(rng, 2, 512 if form == "chunks" else 128)
    return _attend(hq, hkv, d, bf16, page, _log(rng, 1, max(1, 1024 // new_hi)), rng.randint(1, hi), hi, rng.randint(1, new_hi), new_hi,
                   chunked=rng.choice([0, 0, 1]) if form == "wide" else 0)


# ---------------------------------------------------------------------------
# Shapes of a case


def _lengths(case):
    """(cached, new) tokens of every request, always the same for one case; new = -1: ended."""
    r = random.Random(case["requests"] * 1000003 + case["lo"] * 1009 + case["hi"])
    n = case["requests"]
    past = [r.randint(case["lo"], case["hi"]) for _ in range(n)]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(n)]
    for i in range(min(n, case.get("chunked", 0))):
        new[i] = 8 * case["new_hi"]
    return past, [-1 if r.random() < case.get("ended", 0.0) else x for x in new]


def _pages(n, page):
    return -(-n // page)


def _dtype(case):
    return torch.bfloat16 if case["bf16"] else torch.float32


def _seen(case, past, new):
    """(pairs of one query head, keys that some new token of a request sees)."""
    w, s = case["window"], case["sinks"]
    if not w:
        return new * past + new * (new + 1) // 2, past + new
    pairs = sum(min(p + 1, w) + min(s, max(0, p + 1 - w)) for p in range(past, past + new))
    first = max(0, past - w + 1)
    return pairs, past + new - first + min(s, first)


def work(case):
    if case["kind"] == "rope":
        e = 2 if case["bf16"] else 4
        rows = case["hq"] + case["hkv"] * (2 if case["store"] else 1)
        return dict(bytes=2 * case["t"] * rows * case["d"] * e + 8 * case["t"], flops=3.0 * case["t"] * (case["hq"] + case["hkv"]) * case["rotary"])
    past, new = _lengths(case)
    b = f = 0.0
    if case["kind"] in ("tables", "step"):
        t = sum(max(0, n) for n in new)
        moved = sum(_pages(p + n, case["page"]) - _pages(p, case["page"]) if n >= 0 else _pages(p, case["page"]) for p, n in zip(past, new))
        touched = sum(_pages(p + n, case["page"]) - p // case["page"] for p, n in zip(past, new) if n > 0)
        b += 4.0 * (4 * len(new) + 2 * t + 2 * moved + touched)
        f += 4.0 * (len(new) + t)
    if case["kind"] in ("attend", "step"):
        e = 2 if case["bf16"] else 4
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        seen = [_seen(case, p, n) for p, n in zip(past, new)]
        b += e * d * (2.0 * hkv * sum(k for _, k in seen) + 2.0 * hq * sum(new)) + 4.0 * sum(_pages(p + n, case["page"]) for p, n in zip(past, new))
        f += 4.0 * d * hq * sum(p for p, _ in seen)
        if case["kind"] == "step":
            b += e * d * sum(new) * (2.0 * hq + 3.0 * hkv)
            f += 3.0 * d * sum(new) * (hq + hkv)
    return dict(bytes=b, flops=f)


# ---------------------------------------------------------------------------
# Inputs

LINEAR, STRETCH, ORIGINAL = 8.0, 4.0, 32768  # position scalings: factors, and the context that was trained on


def _rot_args(case):
    kind = case.get("scaling", "none")
    args = dict(theta=case.get("theta", 1e6), rotary_dim=case.get("rotary", case["d"]), scaling=kind)
    if kind == "linear":
        args.update(factor=LINEAR)
    elif kind == "yarn":
        args.update(factor=STRETCH, original=ORIGINAL)
    elif kind == "wavelength":
        args.update(factor=STRETCH, original=ORIGINAL, low=1.0, high=4.0)
    return args


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _requests(case, g, dev, s):
    """Cached and new lengths, block tables over shuffled pages, the ring of the free ones."""
    past, new = _lengths(case)
    page = case["page"]
    s["lengths"], s["new"] = _i32(past, dev), _i32(new, dev)
    held = [_pages(p, page) for p in past]
    total = [_pages(p + max(0, n), page) for p, n in zip(past, new)]
    s["t"] = sum(max(0, n) for n in new)
    s["n_pages"] = sum(total) + 7
    s["max_pages"] = max(1, max(total)) + 1
    order = torch.randperm(s["n_pages"], generator=g, device=dev).to(torch.int32)
    table = torch.full((len(past), s["max_pages"]), -1, dtype=torch.int32, device=dev)
    upto = held if case["kind"] in ("tables", "step") else total
    j = torch.arange(s["max_pages"], device=dev)
    counts = torch.tensor(upto, device=dev)
    first = counts.cumsum(0) - counts
    table = torch.where(j < counts[:, None], order[(first[:, None] + j).clamp(max=s["n_pages"] - 1)], table)
    s["block_table"], used = table.contiguous(), sum(upto)
    # the free pages stand in the ring from a place in its middle on
    head = s["n_pages"] // 3
    s["free"] = torch.full((s["n_pages"],), -1, dtype=torch.int32, device=dev)
    s["free"][(head + torch.arange(s["n_pages"] - used, device=dev)) % s["n_pages"]] = order[used:]
    s["ring"] = _i32([head, s["n_pages"] - used, 0, 0], dev)


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case=case)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=dev).to(_dtype(case))  # noqa: E731
    kind = case["kind"]
    if kind == "rope":
        t, d, page = case["t"], case["d"], case["page"]
        s["q"], s["k"] = randn(t, case["hq"], d), randn(t, case["hkv"], d)
        s["pos"] = torch.randint(0, case["far"], (t,), generator=g, device=dev).to(torch.int32)
        if case["store"]:
            s["v"] = randn(t, case["hkv"], d)
            n = _pages(t, page) + 3
            s["slots"] = torch.randperm(n * page, generator=g, device=dev)[:t].to(torch.int32)
            s["k_cache"], s["v_cache"] = (torch.zeros(n, page, case["hkv"], d, dtype=_dtype(case), device=dev) for _ in range(2))
    else:
        _requests(case, g, dev, s)
        r, t = case["requests"], s["t"]
        s["cu"] = torch.zeros(r + 1, dtype=torch.int32, device=dev)
        if kind in ("tables", "step"):
            room = t + 16  # rows of a captured pass that stay empty
            s["pos"], s["slots"] = (torch.zeros(room, dtype=torch.int32, device=dev) for _ in range(2))
            s["lengths_out"], s["ring_out"] = torch.zeros_like(s["lengths"]), torch.zeros_like(s["ring"])
        else:
            room = t
            s["lengths"] = s["lengths"] + s["new"]
            s["cu"][1:] = s["new"].cumsum(0)
        if kind != "tables":
            shape = (s["n_pages"], case["page"], case["hkv"], case["d"])
            s["k_cache"], s["v_cache"] = randn(*shape), randn(*shape)
            s["q"] = randn(room, case["hq"], case["d"])
            if kind == "step":
                s["k"], s["v"] = randn(room, case["hkv"], case["d"]), randn(room, case["hkv"], case["d"])
            s["out"] = torch.zeros_like(s["q"])
    if own:  # what such a program makes once: the angles' table, the attention's workspace
        cev = _cev_hip()
        if kind in ("rope", "step"):
            s["rot"] = cev.RotaryAngles(device=dev, **_rot_args(case))
        if kind in ("attend", "step"):
            s["attention"] = cev.PagedAttention(s["q"], s["k_cache"], s["block_table"], max_new=max(_lengths(case)[1]), window=case["window"],
                                                sinks=case["sinks"])
    elif kind in ("rope", "step"):
        s["inv"], s["factor"] = _inverse_frequencies(_rot_args(case), dev)
    return s


def _inverse_frequencies(a, dev):
    """(angle of each pair per position, the factor on cos and sin), from the scalings' definitions in 64 bits."""
    i = torch.arange(a["rotary_dim"] // 2, dtype=torch.float64, device=dev)
    inv = a["theta"] ** (-2.0 * i / a["rotary_dim"])
    if a["scaling"] == "linear":
        return inv / a["factor"], 1.0
    if a["scaling"] == "yarn":  # pairs of at least 32 turns in the trained context as they are, below one turn stretched, a ramp between
        at = lambda turns: a["rotary_dim"] * math.log(a["original"] / (turns * 2 * math.pi)) / (2 * math.log(a["theta"]))  # noqa: E731
        low, high = max(0, math.floor(at(32.0))), min(a["rotary_dim"] - 1, math.ceil(at(1.0)))
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        return inv / a["factor"] * ramp + inv * (1 - ramp), 0.1 * math.log(a["factor"]) + 1
    if a["scaling"] == "wavelength":  # the same by wavelength
        turns = a["original"] * inv / (2 * math.pi)
        keep = ((turns - a["low"]) / (a["high"] - a["low"])).clamp(0, 1)
        return inv / a["factor"] * (1 - keep) + inv * keep, 1.0
    return inv, 1.0


# ---------------------------------------------------------------------------
# The operators in their plain form


def _plain_tables(s):
    case, page, n_pages = s["case"], s["case"]["page"], s["n_pages"]
    length, new = s["lengths"].long(), s["new"].long()
    ended, add = new < 0, new.clamp(min=0)
    have = (length + page - 1) // page
    need = torch.where(ended, 0, (length + add + page - 1) // page - have)
    give = torch.where(ended, have, 0)
    head, count = s["ring"][0].long(), s["ring"][1].long()
    j = torch.arange(s["max_pages"], device=length.device)
    taken = (head + (need.cumsum(0) - need)[:, None] + j - have[:, None]) % n_pages
    fresh = (j >= have[:, None]) & (j < (have + need)[:, None])
    back = j < give[:, None]
    place = torch.where(back, (head + count + (give.cumsum(0) - give)[:, None] + j) % n_pages, n_pages)
    ring = torch.cat([s["free"], s["free"][:1]])
    ring = ring.scatter(0, place.reshape(-1), s["block_table"].reshape(-1))[:n_pages]
    s["block_table"].copy_(torch.where(fresh, s["free"][taken], s["block_table"]))
    s["free"].copy_(ring)
    s["cu"][1:] = add.cumsum(0)
    i = torch.arange(s["pos"].shape[0], device=length.device)
    r = torch.searchsorted(s["cu"][1:].long(), i, right=True).clamp(max=case["requests"] - 1)
    real = i < s["cu"][-1]
    pos = torch.where(real, length[r] + i - s["cu"][r], 0)
    slots = torch.where(real, s["block_table"][r, pos // page].long() * page + pos % page, -1)
    s["pos"].copy_(pos)
    s["slots"].copy_(slots)
    s["lengths_out"].copy_(torch.where(ended, 0, length + add))
    zero = torch.zeros_like(head)
    s["ring_out"].copy_(torch.stack([(head + need.sum()) % n_pages, count - need.sum() + give.sum(), zero, zero]))


def _rotate(x, cos, sin, rotary, interleaved):
    a, rest = x[..., :rotary].float(), x[..., rotary:].float()
    a, b = (a[..., 0::2], a[..., 1::2]) if interleaved else (a[..., : rotary // 2], a[..., rotary // 2:])
    y, z = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([y, z], -1).flatten(-2) if interleaved else torch.cat([y, z], -1)
    return torch.cat([y, rest], -1).to(x.dtype)


def _plain_rope(s, q_out=None):
    case = s["case"]
    rotary, interleaved = case.get("rotary", case["d"]), case.get("interleaved", False)
    angle = s["pos"].double()[:, None, None] * s["inv"]
    cos, sin = (s["factor"] * angle.cos()).float(), (s["factor"] * angle.sin()).float()
    if not case.get("store", True):
        sin = -sin
    q, k = (_rotate(x, cos, sin, rotary, interleaved) for x in (s["q"], s["k"]))
    if "slots" in s:
        rows = lambda cache: cache.view(-1, *cache.shape[2:])  # noqa: E731
        at = s["slots"].long()
        if case["kind"] == "step":  # rows of no request are stored nowhere
            at = at[: s["t"]]
        rows(s["k_cache"])[at] = k[: at.shape[0]]
        rows(s["v_cache"])[at] = s["v"][: at.shape[0]]
    return q, k


def _plain_attend(s, q, lengths):
    case, dev = s["case"], q.device
    hq, hkv, d, r = case["hq"], case["hkv"], case["d"], case["requests"]
    n_max, page = max(1, max(_lengths(case)[1])), case["page"]
    cu = s["cu"].long()
    count = cu[1:] - cu[:-1]
    i = torch.arange(n_max, device=dev)
    rows = (cu[:-1, None] + i).clamp(max=s["t"] - 1)
    pos = lengths.long()[:, None] - count[:, None] + i                       # (r, n)
    qs = q[rows].float().view(r, n_max, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(r * hkv, -1, d)

    def gathered(cache):  # (r, hkv, keys, d)
        x = cache[s["block_table"][:, : s["max_pages"] - 1].long().clamp(min=0)]
        return x.flatten(1, 2).permute(0, 2, 1, 3).float().reshape(r * hkv, -1, d)

    k, v = gathered(s["k_cache"]), gathered(s["v_cache"])
    key = torch.arange(k.shape[1], device=dev)
    seen = key <= pos[..., None]
    if case["window"]:
        seen &= (key > pos[..., None] - case["window"]) | (key < case["sinks"])
    score = torch.bmm(qs, k.transpose(1, 2).contiguous()).mul_(1 / math.sqrt(d)).view(r, hkv, hq // hkv, n_max, -1)
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.reshape(r * hkv, -1, k.shape[1]), v).view(r, hkv, hq // hkv, n_max, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(r, n_max, hq, d).to(q.dtype)
    # rows past a request's own go to a row behind all of them
    at = torch.where(i < count[:, None], rows, s["out"].shape[0])
    grown = torch.cat([s["out"], s["out"][:1]])
    grown[at.reshape(-1)] = o.reshape(-1, hq, d)
    s["out"].copy_(grown[:-1])


def _tables_out(s):
    return {k: s[k] for k in ("lengths_out", "ring_out", "block_table", "free", "cu", "pos", "slots")}


def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if own:
        cev = _cev_hip()
        if kind in ("tables", "step"):
            cev.paged_tables(s["lengths"], s["new"], s["block_table"], case["page"], s["cu"], s["pos"], s["slots"], free=s["free"],
                             ring=s["ring"], lengths_out=s["lengths_out"], ring_out=s["ring_out"])
            if kind == "tables":
                return _tables_out(s)
        if kind == "rope":
            if not case["store"]:
                q, k = cev.rope(s["q"], s["k"], s["pos"], s["rot"], interleaved=case["interleaved"], transposed=True)
                return {"q": q, "k": k}
            q, _, _ = cev.rope(s["q"], s["k"], s["pos"], s["rot"], interleaved=case["interleaved"], v_in=s["v"], k_out=s["k_cache"],
                            v_out=s["v_cache"], slots=s["slots"])
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        q, lengths = s["q"], s["lengths"]
        if kind == "step":
            q, _, _ = cev.rope(q, s["k"], s["pos"], s["rot"], v_in=s["v"], k_out=s["k_cache"], v_out=s["v_cache"], slots=s["slots"])
            lengths = s["lengths_out"]
        attention = s["attention"]
        attention.plan(s["cu"], lengths)
        attention(q, s["k_cache"], s["v_cache"], s["block_table"], out=s["out"])
    else:
        if kind in ("tables", "step"):
            _plain_tables(s)
            if kind == "tables":
                return _tables_out(s)
        if kind == "rope":
            q, k = _plain_rope(s)
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]} if case["store"] else {"q": q, "k": k}
        q, lengths = s["q"], s["lengths"]
        if kind == "step":
            q, _ = _plain_rope(s)
            lengths = s["lengths_out"]
        _plain_attend(s, q, lengths)
    if kind == "step":
        return dict(_tables_out(s), out=s["out"], k_cache=s["k_cache"], v_cache=s["v_cache"])
    return s["out"]


# ---------------------------------------------------------------------------
# The operators from their definitions in 64 bits


def _exact_tables(s):
    """One request after the other, on the host."""
    page, n_pages = s["case"]["page"], s["n_pages"]
    length, new, table, free = (s[k].tolist() for k in ("lengths", "new", "block_table", "free"))
    head, count = s["ring"].tolist()[:2]
    tail, first_tail = head + count, head + count
    cu, pos, slots = [0], [], []
    for r, n in enumerate(new):
        if n < 0:
            for j in range(_pages(length[r], page)):
                free[tail % n_pages] = table[r][j]
                tail += 1
            length[r], n = 0, 0
        for p in range(length[r], length[r] + n):
            if p % page == 0:
                table[r][p // page] = free[head % n_pages]
                head += 1
            pos.append(p)
            slots.append(table[r][p // page] * page + p % page)
        length[r] += n
        cu.append(len(pos))
    assert head <= first_tail
    spare = s["pos"].shape[0] - len(pos)
    dev = s["lengths"].device
    return {k: _i32(v, dev) for k, v in dict(lengths_out=length, ring_out=[head % n_pages, tail - head, 0, 0], block_table=table, free=free, cu=cu,
                                             pos=pos + [0] * spare, slots=slots + [-1] * spare).items()}


def _exact_turns(a):
    """Pair by pair: the angle per position, and the factor on the rotated values."""
    found = []
    for i in range(a["rotary_dim"] // 2):
        inv = math.exp(-2.0 * i / a["rotary_dim"] * math.log(a["theta"]))
        if a["scaling"] == "none":
            share = 0.0  # of the stretched angle
        elif a["scaling"] == "linear":
            share = 1.0
        elif a["scaling"] == "wavelength":
            turns = a["original"] * inv / (2 * math.pi)
            share = 1 - min(1.0, max(0.0, (turns - a["low"]) / (a["high"] - a["low"])))
        else:
            # the pair whose wavelength fits `turns` times into the trained context
            pair = lambda turns: math.log(a["original"] / (2 * math.pi * turns), a["theta"]) * a["rotary_dim"] / 2  # noqa: E731
            low, high = max(0, math.floor(pair(32))), min(a["rotary_dim"] - 1, math.ceil(pair(1)))
            share = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
        found.append(inv * (1 - share + share / a.get("factor", 1.0)))
    return found, 1 + 0.1 * math.log(a["factor"]) if a["scaling"] == "yarn" else 1.0


def _exact_rope(x, s, inv, factor, sign):
    """Pairs as complex numbers, turned by their angle."""
    case = s["case"]
    rotary = case.get("rotary", case["d"])
    y = x.double().clone()
    turn = torch.polar(torch.full_like(inv, factor).expand(s["pos"].shape[0], -1), sign * s["pos"].double()[:, None] * inv)[:, None]
    first = torch.arange(0, rotary, 2) if case.get("interleaved", False) else torch.arange(rotary // 2)
    second = first + (1 if case.get("interleaved", False) else rotary // 2)
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_store(s, cache, rows, slots):
    c = s[cache].double().clone()
    page = s["case"]["page"]
    c[slots // page, slots % page] = rows.double()
    return c


def _exact_attend(s, q, k_cache, v_cache, table, past, new):
    """Request after request, 256 rows at a time."""
    case = s["case"]
    g, page = case["hq"] // case["hkv"], case["page"]
    out, row = s["out"].double().clone(), 0
    for r, (p, n) in enumerate(zip(past, new)):
        pages = table[r, : _pages(p + n, page)].long()
        k, v = (c[pages].flatten(0, 1)[: p + n].double().permute(1, 0, 2) for c in (k_cache, v_cache))
        for a in range(0, n, 256):
            b = min(n, a + 256)
            x = q[row + a: row + b].double().view(b - a, case["hkv"], g, -1).permute(1, 2, 0, 3).reshape(case["hkv"], g * (b - a), -1)
            score = (x @ k.transpose(1, 2).contiguous()).view(case["hkv"], g, b - a, -1) / math.sqrt(case["d"])
            ahead = torch.arange(p + n, device=q.device) - torch.arange(p + a, p + b, device=q.device)[:, None]
            hidden = ahead > 0
            if case["window"]:
                hidden |= (ahead <= -case["window"]) & (torch.arange(p + n, device=q.device) >= case["sinks"])
            weight = torch.softmax(score.masked_fill(hidden, float("-inf")), -1)
            o = (weight.view(case["hkv"], g * (b - a), -1) @ v).view(case["hkv"], g, b - a, -1)
            out[row + a: row + b] = o.permute(2, 0, 1, 3).reshape(b - a, case["hq"], -1)
        row += n
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kind = case["kind"]
    if kind in ("rope", "step"):
        inv, factor = _exact_turns(_rot_args(case))
        inv = torch.tensor(inv, dtype=torch.float64, device=s["q"].device)
    if kind in ("tables", "step"):
        found = _exact_tables(s)
        if kind == "tables":
            return found
        s["pos"], s["slots"], s["block_table"] = found["pos"], found["slots"], found["block_table"]
    if kind in ("rope", "step"):
        sign = 1.0 if case.get("store", True) else -1.0
        q, k = (_exact_rope(s[x], s, inv, factor, sign) for x in "qk")
        if sign < 0:
            return {"q": q, "k": k}
        n = s["t"] if kind == "step" else case["t"]
        at = s["slots"][:n].long()
        kc, vc = _exact_store(s, "k_cache", k[:n], at), _exact_store(s, "v_cache", s["v"][:n], at)
        if kind == "rope":
            return {"q": q, "k_cache": kc, "v_cache": vc}
        # the attention reads what the model's type holds
        dt = _dtype(case)
        out = _exact_attend(s, q.to(dt), kc.to(dt), vc.to(dt), s["block_table"], *_lengths(case))
        return dict(found, out=out, k_cache=kc, v_cache=vc)
    return _exact_attend(s, s["q"], s["k_cache"], s["v_cache"], s["block_table"], *_lengths(case))
