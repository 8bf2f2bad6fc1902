"""Serving over a paged cache: page tables, rotary positions, attention over
pages, each against a plain implementation in 64 bits, and a run of them
together.  The host side and every refusal are tested on the CPU."""
import ctypes as C
import math
import random

import numpy as np
import pytest

import cev_hip
from cev_hip import CevError, _abi

# Half a step of each type's rounding, relative to the value.
HALF = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def _torch_type(name):
    import torch
    return {"bf16": torch.bfloat16, "f32": torch.float32}[name]


# ---------------------------------------------------------------------------
# Host side


def _paged_desc(hq=8, hkv=2, d=128, requests=3, t=40, page=16, n_pages=50, max_pages=10, dtype=_abi.CEV_BF16, **kw):
    x = _abi.PagedDesc()
    assert _abi.lib().cev_paged_desc_init(C.byref(x), dtype, hq, hkv, d, requests, t, page, n_pages, max_pages) == 0
    for k, v in kw.items():
        setattr(x, k, v)
    return x


def _work_size(d):
    n = C.c_size_t()
    return _abi.lib().cev_paged_work_size(C.byref(d), C.byref(n)), n.value


def test_paged_desc_layout(cev):
    d = _paged_desc()
    assert (d.q_stride_t, d.q_stride_h) == (1024, 128) and (d.kc_stride_p, d.kc_stride_t, d.kc_stride_h) == (16 * 256, 256, 128)
    assert d.max_new == 40 and d.bt_stride == 10 and np.float32(d.scale) == np.float32(1 / np.sqrt(128))
    rc, n = _work_size(d)
    assert rc == 0 and n > 0
    assert _abi.lib().cev_paged_work_size(None, C.byref(C.c_size_t())) == -1 and _abi.lib().cev_paged_work_size(C.byref(d), None) == -1


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=7), -2), (dict(d=64), -2), (dict(d=256, dtype=_abi.CEV_F32), -2), (dict(hq=6), -2), (dict(hq=7), -1), (dict(hq=0), -1),
    (dict(requests=0), -1), (dict(requests=5000), -2), (dict(t=0), -1), (dict(max_new=0), -1), (dict(max_new=41), -1),
    (dict(page=8), -1), (dict(page=48), -1), (dict(page=2048), -1), (dict(n_pages=0), -1), (dict(max_pages=0), -1),
    (dict(max_pages=1 << 27), -1), (dict(window=-1), -1), (dict(window=4, sinks=-1), -1), (dict(sinks=4), -1),
    (dict(scale=0.0), -1), (dict(scale=math.inf), -1), (dict(scale=math.nan), -1), (dict(q_stride_h=100), -2), (dict(kc_stride_p=-8), -1),
    (dict(kc_stride_t=120), -2), (dict(vc_stride_t=1 << 40), -2), (dict(o_stride_t=1 << 62), -1), (dict(bt_stride=9), -1),
])
def test_paged_descriptors_out_of_bounds_are_refused(cev, kw, code):
    assert _work_size(_paged_desc(**kw))[0] == code
    assert _abi.lib().cev_last_error()


@pytest.mark.parametrize("kw", [dict(o_stride_t=0), dict(o_stride_h=64), dict(o_stride_h=0)])
def test_overlapping_rows_of_out_are_refused(cev, kw):
    assert _work_size(_paged_desc(**kw))[0] == -1


def test_strides_of_single_rows_do_not_count(cev):
    """A tensor's stride over a dimension of size one may be anything."""
    assert _work_size(_paged_desc(t=1, q_stride_t=3, o_stride_t=1))[0] == 0
    assert _work_size(_paged_desc(hq=1, hkv=1, q_stride_h=1, o_stride_h=0, kc_stride_h=5, vc_stride_h=1))[0] == 0
    assert _work_size(_paged_desc(n_pages=1, kc_stride_p=1, vc_stride_p=7))[0] == 0


def test_paged_calls_check_their_buffers(cev):
    L, d = _abi.lib(), _paged_desc()
    n = _work_size(d)[1]
    fake = lambda a=4096: C.c_void_p(a)  # noqa: E731  (refused before anything reads it)
    assert L.cev_paged_plan(C.byref(d), None, fake(), fake(), n, None) == -1
    assert L.cev_paged_plan(C.byref(d), fake(), fake(), fake(4100), n, None) == -1
    assert L.cev_paged_plan(C.byref(d), fake(), fake(), fake(), n - 1, None) == -4
    ok = [fake()] * 6
    for i in range(6):
        bad = list(ok)
        bad[i] = None
        assert L.cev_paged_attention(C.byref(d), *bad, n, None) == -1
        bad[i] = fake(4098)
        assert L.cev_paged_attention(C.byref(d), *bad, n, None) == -1
    assert L.cev_paged_attention(C.byref(d), *ok, n - 1, None) == -4
    args = [3, 16, 50, 10, 40, *[fake()] * 3, 10, *[fake()] * 7, None]
    for i, v, code in ((0, 0, -1), (0, 4097, -2), (1, 24, -1), (1, 0, -1), (2, 0, -1), (3, 0, -1), (4, -1, -1), (2, 1 << 28, -1),
                       (3, 1 << 27, -1), (8, 9, -1), (5, None, -1), (6, None, -1), (7, None, -1), (10, None, -1), (11, None, -1),
                       (12, None, -1), (13, None, -1), (14, None, -1), (15, None, -1)):
        bad = list(args)
        bad[i] = v
        assert L.cev_paged_tables(*bad) == code, (i, v)


def _rope_desc(**kw):
    d = _abi.RopeDesc()
    assert _abi.lib().cev_rope_desc_init(C.byref(d), _abi.CEV_BF16, 8, 2, 128, 5, 128, 16, 160) == 0
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_rope_calls_are_checked(cev):
    L = _abi.lib()
    fake = C.c_void_p(4096)
    ok = [fake] * 9  # q k v pos steps slots q_out k_out v_out
    run = lambda d, p: L.cev_rope(C.byref(d), *p, None)  # noqa: E731
    for kw, code in ((dict(dtype=3), -2), (dict(head_dim=120), -2), (dict(head_dim=272), -2), (dict(rotary_dim=0), -2),
                     (dict(rotary_dim=136), -2), (dict(rotary_dim=144), -2), (dict(t=-1), -1), (dict(n_q_heads=-1), -1),
                     (dict(n_kv_heads=40000), -1), (dict(factor=math.nan), -1), (dict(factor=math.inf), -1), (dict(qi_stride_t=-8), -1),
                     (dict(ko_stride_h=4), -2), (dict(page_size=24), -1), (dict(n_slots=-1), -1)):
        assert run(_rope_desc(**kw), ok) == code, kw
    for i in (0, 1, 2, 3, 4, 6, 7, 8):  # v_in without v_out and the other way round, too
        bad = list(ok)
        bad[i] = None
        assert run(_rope_desc(), bad) == -1, i
    for i, at in ((0, 4104), (3, 4098), (4, 4100), (5, 4098), (8, 4104)):
        bad = list(ok)
        bad[i] = C.c_void_p(at)
        assert run(_rope_desc(), bad) == -1, i
    assert L.cev_rope(None, *ok, None) == -1
    assert run(_rope_desc(t=0), [None] * 9) == 0 and run(_rope_desc(n_q_heads=0, n_kv_heads=0), [None] * 9) == 0


@pytest.mark.parametrize("kw", [dict(qo_stride_t=0), dict(qo_stride_h=64), dict(ko_stride_h=64), dict(vo_stride_t=0), dict(vo_stride_p=0),
                                dict(ko_stride_p=64)])
def test_overlapping_rows_of_rope_are_refused(cev, kw):
    ok = [C.c_void_p(4096)] * 9
    assert _abi.lib().cev_rope(C.byref(_rope_desc(**kw)), *ok, None) == -1


@pytest.mark.parametrize("scaling,args", [("none", {}), ("linear", dict(factor=8.0)), ("yarn", dict(factor=4.0, original=32768)),
                                          ("yarn", dict(factor=16.0, original=4096, low=2.0, high=20.0, attention_factor=1.25)),
                                          ("wavelength", dict(factor=8.0, original=8192))])
@pytest.mark.parametrize("rotary_dim,theta", [(128, 1e6), (64, 1e7), (16, 10000.0)])
def test_rotary_angles(cev, scaling, args, rotary_dim, theta):
    """The steps against the scalings' definitions: half a step of 2^-64 turns, and 2^-50 of the value for this formula's 64 bits."""
    rot = cev.RotaryAngles(theta, rotary_dim, "cpu", scaling=scaling, **args)
    f, original = args.get("factor", 1.0), args.get("original", 0.0)
    low, high = args.get("low", 1.0), args.get("high", 4.0 if scaling == "wavelength" else 32.0)
    pair = lambda n: rotary_dim * math.log(original / (2 * math.pi * n)) / (2 * math.log(theta))  # noqa: E731
    for i, got in enumerate(rot.turns):
        inv = theta ** (-2 * i / rotary_dim)
        if scaling == "none":
            want = inv
        elif scaling == "linear":
            want = inv / f
        elif scaling == "yarn":
            a, b = max(0, math.floor(pair(high))), min(rotary_dim - 1, math.ceil(pair(low)))
            r = min(1.0, max(0.0, (i - a) / max(b - a, 1e-3)))
            want = inv / f * r + inv * (1 - r)
        else:
            wave = 2 * math.pi / inv
            if wave < original / high:
                want = inv
            elif wave > original / low:
                want = inv / f
            else:
                s = (original / wave - low) / (high - low)
                want = (1 - s) * inv / f + s * inv
        assert abs(got / 2.0 ** 64 * 2 * math.pi - want) <= 2.0 ** -50 * inv + math.pi * 2.0 ** -64
    assert rot.factor == pytest.approx(args.get("attention_factor", 0.1 * math.log(f) + 1 if scaling == "yarn" else 1.0), rel=1e-7)
    signed = rot.steps.tolist()
    assert [x % (1 << 64) for x in signed] == rot.turns


@pytest.mark.parametrize("kw,code", [
    (dict(theta=1.0), -1), (dict(theta=math.nan), -1), (dict(theta=math.inf), -1), (dict(rotary_dim=0), -1), (dict(rotary_dim=7), -1),
    (dict(rotary_dim=1 << 33), -1), (dict(scaling="other"), -2), (dict(scaling="linear", factor=0.5), -1), (dict(scaling="linear", factor=math.nan), -1),
    (dict(scaling="yarn", factor=2.0), -1), (dict(scaling="yarn", factor=2.0, original=100, low=3.0, high=3.0), -1),
    (dict(scaling="wavelength", factor=2.0, original=math.inf), -1), (dict(attention_factor=-1.0), -1),
])
def test_rotary_angles_refuse(cev, kw, code):
    with pytest.raises(CevError) as e:
        cev.RotaryAngles(**dict(dict(theta=1e6, rotary_dim=64, device="cpu"), **kw))
    assert e.value.code == code


def test_paged_python_calls_check_tensors(cev):
    """What the calls can tell from shapes and types is refused before a device is looked at; then CPU tensors are."""
    import torch
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt)  # noqa: E731
    i = lambda *s: z(*s, dt=torch.int32)  # noqa: E731

    def refused(match, code, fn, *a, **kw):
        with pytest.raises(CevError, match=match) as e:
            fn(*a, **kw)
        assert e.value.code == code

    tables = dict(lengths=i(3), new_len=i(3), block_table=i(3, 4), page_size=16, cu=i(4), pos=i(10), slots=i(10), free=i(20), ring=i(4))
    for name, bad in (("new_len", i(2)), ("lengths", i(3).long()), ("lengths", i(3, 1)), ("block_table", i(2, 4)), ("block_table", i(3, 8)[:, ::2]),
                      ("cu", i(3)), ("slots", i(9)), ("ring", i(3)), ("free", i(20).long()), ("lengths_out", i(4)), ("ring_out", i(5)),
                      ("pos", i(20)[::2]), ("page_size", 1 << 40), ("ring", None), ("n_pages", 19)):
        refused("", -1, cev.paged_tables, **dict(tables, **{name: bad}))
    refused("required", -1, cev.paged_tables, **dict(tables, free=None))
    refused("must be on the GPU", -1, cev.paged_tables, **tables)

    rot = cev.RotaryAngles(1e6, 128, "cpu")
    q, k, pos = z(5, 4, 128), z(5, 2, 128), i(5)
    kc = z(3, 16, 2, 128)
    refused("shar", -1, cev.rope, q, k.bfloat16(), pos, rot)
    refused("float16", -2, cev.rope, q.half(), k.half(), pos, rot)
    refused("k_in", -1, cev.rope, q, k[:4], pos, rot)
    refused("pos", -1, cev.rope, q, k, pos.long(), rot)
    refused("pos", -1, cev.rope, q, k, i(4), rot)
    refused("q_out", -1, cev.rope, q, k, pos, rot, q_out=q[:, :3])
    refused("k_out", -1, cev.rope, q, k, pos, rot, k_out=z(4, 2, 128))
    refused("caches", -1, cev.rope, q, k, pos, rot, slots=i(5))
    refused("caches", -1, cev.rope, q, k, pos, rot, slots=i(5), k_out=kc, v_in=k)
    refused("caches", -1, cev.rope, q, k, pos, rot, slots=i(5), k_out=kc, v_in=k, v_out=z(2, 16, 2, 128))
    refused("slots", -1, cev.rope, q, k, pos, rot, slots=i(6), k_out=kc)
    refused("v_in", -1, cev.rope, q, k, pos, rot, v_in=z(5, 3, 128))
    refused("contiguous", -2, cev.rope, z(5, 128, 4).transpose(1, 2), k, pos, rot)
    refused("must be on the GPU", -1, cev.rope, q, k, pos, rot)

    bt = i(2, 4)
    for bad in (dict(window=1 << 32), dict(max_new=6), dict(sinks=3), dict(scale=0.0), dict(max_new=(1 << 32) + 1)):
        refused("", -1, cev.PagedAttention, q, kc, bt, **bad)
    refused("share", -1, cev.PagedAttention, q, kc.bfloat16(), bt)
    refused("not supported", -2, cev.PagedAttention, q.double(), kc.double(), bt)
    refused("must be", -1, cev.PagedAttention, q[0], kc, bt)
    att = cev.PagedAttention(q, kc, bt)
    refused("cu", -1, att.plan, i(2), i(2))
    refused("lengths", -1, att.plan, i(3), i(2).long())
    refused("must be on the GPU", -1, att.plan, i(3), i(2))
    refused("q and out", -1, att, z(4, 4, 128), kc, kc, bt)
    refused("caches", -1, att, q, kc, z(4, 16, 2, 128), bt)
    refused("type", -1, att, q, kc, kc.bfloat16(), bt)
    refused("entries", -1, att, q, kc, kc, i(2, 5))
    refused("block_table", -1, att, q, kc, kc, i(3, 4))
    refused("contiguous", -2, att, q, kc.transpose(2, 3).contiguous().transpose(2, 3), kc, bt)
    refused("must be on the GPU", -1, att, q, kc, kc, bt)


# ---------------------------------------------------------------------------
# Page tables


def _tables_oracle(lengths, new, table, free, ring, page, n_pages, max_tokens):
    """One request after the other: the definition."""
    lengths, table = list(lengths), [list(r) for r in table]
    max_pages = len(table[0])
    pages = lambda n: -(-n // page)  # noqa: E731
    status = 0
    for n, a in zip(lengths, new):
        if not 0 <= n <= max_pages * page or a < -1:
            status |= 8
        elif a > max_pages * page - n:
            status |= 2
    cu, pos, slots, given, taken = [0], [], [], [], 0
    fresh = list(free) if free is not None else None
    if not status:
        head, count = ring[:2]
        for r, a in enumerate(new):
            if a < 0:
                if free is not None:
                    given += table[r][: pages(lengths[r])]
                lengths[r] = 0
            for p in range(lengths[r], lengths[r] + max(0, a)):
                if free is not None and p % page == 0:
                    table[r][p // page] = free[(head + taken) % n_pages] if taken < count else None
                    taken += 1
                e = table[r][p // page]
                pos.append(p)
                slots.append(-1 if e is None or not 0 <= e < n_pages else e * page + p % page)
            lengths[r] += max(0, a)
            cu.append(len(pos))
        if len(pos) > max_tokens:
            status |= 1
        if free is not None and taken > count:
            status |= 4
        if not status and free is not None:
            for i, e in enumerate(given):
                fresh[(head + count + i) % n_pages] = e
    if status:
        return dict(status=status)
    ring = [(ring[0] + taken) % n_pages, ring[1] - taken + len(given), 0, 0] if free is not None else [ring[0], ring[1], 0, 0]
    pad = max_tokens - len(pos)
    return dict(status=0, lengths=lengths, table=table, free=fresh, ring=ring, cu=cu, pos=pos + [0] * pad, slots=slots + [-1] * pad)


class _Tables:
    """Requests with shuffled pages on the device."""

    def __init__(self, dev, lengths, page, max_pages, spare, seed, max_tokens, extra_stride=0):
        import torch
        rng = random.Random(seed)
        held = [-(-n // page) for n in lengths]
        self.n_pages = max(1, sum(held) + spare)
        order = list(range(self.n_pages))
        rng.shuffle(order)
        self.table_np, at = [], 0
        for h in held:
            self.table_np.append(order[at: at + h] + [-7] * (max_pages - h))
            at += h
        head = rng.randrange(self.n_pages)
        self.free_np = [-9] * self.n_pages
        for i, e in enumerate(order[at:]):
            self.free_np[(head + i) % self.n_pages] = e
        self.ring_np = [head, self.n_pages - at, 0, 0]
        self.lengths_np, self.page, self.max_tokens = list(lengths), page, max_tokens
        t = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        self.lengths, self.free, self.ring = t(self.lengths_np), t(self.free_np), t(self.ring_np)
        self.table = torch.full((len(lengths), max_pages + extra_stride), -7, dtype=torch.int32, device=dev)[:, :max_pages]
        self.table.copy_(t(self.table_np))
        self.cu = t([-5] * (len(lengths) + 1))
        self.pos, self.slots = t([-5] * max_tokens), t([-5] * max_tokens)
        self.t = t

    def step(self, new, in_place=True, free=True, stream=None):
        import torch
        lo, ro = (None, None) if in_place else (torch.full_like(self.lengths, -5), self.t([-5, -5, -5, 0]))
        cev_hip.paged_tables(self.lengths, self.t(new), self.table, self.page, self.cu, self.pos, self.slots, free=self.free if free else None,
                             ring=self.ring, n_pages=self.n_pages, lengths_out=lo, ring_out=ro, stream=stream)
        torch.cuda.synchronize()
        if not in_place:
            self.lengths, self.ring = lo, ro

    def check(self, want, what=""):
        assert self.ring.tolist()[2] == want["status"], what
        if want["status"]:
            assert self.cu.tolist() == [0] * len(self.cu) and set(self.slots.tolist()) <= {-1} and set(self.pos.tolist()) <= {0}, what
            assert self.lengths.tolist() == self.lengths_np and self.table.tolist() == self.table_np and self.free.tolist() == self.free_np, what
            assert self.ring.tolist()[:2] == self.ring_np[:2] and self.ring.tolist()[3] == 0
            return
        got = dict(lengths=self.lengths.tolist(), table=self.table.tolist(), ring=self.ring.tolist(), cu=self.cu.tolist(), pos=self.pos.tolist(),
                   slots=self.slots.tolist(), free=self.free.tolist())
        for k, v in got.items():
            if want[k] is not None:
                assert v == want[k], (what, k)
        self.lengths_np, self.table_np, self.ring_np = want["lengths"], want["table"], want["ring"]
        self.free_np = want["free"] if want["free"] is not None else self.free_np

    def expect(self, new, free=True):
        return _tables_oracle(self.lengths_np, new, self.table_np, self.free_np if free else None, self.ring_np, self.page, self.n_pages,
                              self.max_tokens)


@pytest.mark.gpu
@pytest.mark.parametrize("requests,page,longest,new_hi,room", [
    (1, 16, 40, 1, 0), (3, 16, 50, 1, 5), (5, 1, 9, 6, 0), (7, 32, 100, 90, 33), (64, 16, 300, 3, 0), (513, 16, 90, 20, 7), (4096, 4, 30, 5, 100),
    (600, 16, 200, 64, 3)])
@pytest.mark.parametrize("in_place", [True, False])
def test_tables_follow_the_requests(gpu, requests, page, longest, new_hi, room, in_place):
    """Several steps of growing, pausing and ending requests, the pages of
    ended ones among the free ones of later steps."""
    rng = random.Random(requests * 31 + page)
    lengths = [rng.choice([0, rng.randint(0, longest), page * rng.randint(0, longest // page)]) for _ in range(requests)]
    steps = 4
    top = max(lengths) + steps * new_hi
    tokens = requests * new_hi + room
    s = _Tables(gpu, lengths, page, -(-top // page) + 1, requests * (steps * new_hi // page + steps) + 2, seed=requests, max_tokens=tokens, extra_stride=3)
    for k in range(steps):
        new = [rng.choice([-1, 0, 1, rng.randint(0, new_hi), new_hi]) for _ in range(requests)]
        want = s.expect(new)
        assert want["status"] == 0
        s.step(new, in_place)
        s.check(want, f"step {k}")


@pytest.mark.gpu
def test_tables_without_a_ring(gpu):
    """The block table holds the new tokens' pages already; entries out of range give no slot."""
    s = _Tables(gpu, [5, 0, 16], 16, 4, 9, seed=1, max_tokens=70)
    table = [[3, 4, -7, -7], [9, 1, 2, 77], [0, 5, -1, -7]]
    s.table.copy_(s.t(table))
    s.table_np = table
    s.n_pages = 10
    want = s.expect([20, 30, 18], free=False)
    assert -1 in want["slots"][:68]
    s.step([20, 30, 18], free=False)
    s.check(want)


@pytest.mark.gpu
@pytest.mark.parametrize("what,new,change,status", [
    ("tokens", [30, 30, 30], {}, 1), ("length", [0, 10 ** 6, 0], {}, 2), ("length", [2 ** 31 - 1, 2 ** 31 - 1, 0], {}, 2),
    ("pages", [40, 0, 0], dict(ring=[0, 1, 0, 0]), 4), ("new", [0, -2, 0], {}, 8), ("negative", [0, 0, 1], dict(lengths=[5, -1, 3]), 8),
    ("too long", [0, 0, 1], dict(lengths=[5, 10 ** 9, 3]), 8), ("head", [1, 1, 1], dict(ring=[-1, 3, 0, 0]), 8),
    ("head", [1, 1, 1], dict(ring=[10 ** 9, 3, 0, 0]), 8), ("count", [1, 1, 1], dict(ring=[0, 10 ** 9, 0, 0]), 8),
    ("count", [1, 1, 1], dict(ring=[0, -3, 0, 0]), 8), ("given back twice", [-1, 1, 1], dict(ring=[0, -1, 0, 0]), 8)])
def test_tables_out_of_bounds_leave_everything_and_say_so(gpu, what, new, change, status):
    s = _Tables(gpu, [5, 20, 33], 16, 8, 12, seed=2, max_tokens=48)
    if what == "given back twice":
        change = dict(ring=[0, s.n_pages, 0, 0])
    for k, v in change.items():
        getattr(s, k).copy_(s.t(v))
        setattr(s, k + "_np", v)
    if what == "tokens":
        s.max_tokens = 48
    s.step(new)
    s.check(dict(status=status), what)


# ---------------------------------------------------------------------------
# Rotary positions


def _rope_oracle(x, pos, rot, interleaved, transposed):
    """Pairs as complex numbers in 64 bits, angles from the exact fractions of a turn."""
    import torch
    y = x.double().cpu().clone()
    half = rot.rotary_dim // 2
    part = torch.tensor([[((p * s) % (1 << 64)) / 2.0 ** 64 for s in rot.turns] for p in pos.tolist()], dtype=torch.float64)
    angle = 2 * math.pi * part * (-1 if transposed else 1)
    turn = torch.polar(torch.full_like(angle, rot.factor), angle)[:, None]
    first = torch.arange(0, 2 * half, 2) if interleaved else torch.arange(half)
    second = first + (1 if interleaved else half)
    z = torch.complex(y[..., first], y[..., second]) * turn
    size = y.abs()
    size[..., first] = size[..., second] = abs(rot.factor) * torch.hypot(y[..., first], y[..., second])
    y[..., first], y[..., second] = z.real, z.imag
    return y, size


def _rope_close(got, want, size, kind):
    """cos and sin are within 2^-23 (their polynomials 2^-25, the rounded
    angle 2^-25, four roundings of the sums at 2^-25 each), their products
    with the factor and the pair rounded three times more: 2^-21 of the pair's
    size, and half a step of the value in the type."""
    err = (got.double().cpu() - want).abs()
    assert bool((err <= HALF[kind] * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -21 * size + 1e-40).all()), float((err / size.clamp(min=1e-30)).max())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("t,hq,hkv,d,rotary,interleaved", [
    (1, 16, 8, 128, 128, False), (3, 4, 2, 128, 32, True), (17, 3, 1, 80, 48, False), (33, 8, 8, 256, 64, True), (130, 2, 2, 256, 256, False),
    (700, 5, 3, 64, 64, True), (2, 0, 4, 128, 64, False), (5, 4, 0, 16, 16, True), (1500, 32, 8, 128, 128, False)])
def test_rope_matches_64_bits(gpu, kind, t, hq, hkv, d, rotary, interleaved):
    import torch
    g = torch.Generator().manual_seed(t * 7 + d)
    dt = _torch_type(kind)
    rot = cev_hip.RotaryAngles(1e6, rotary, gpu, scaling="yarn", factor=4.0, original=32768)
    q, k = (torch.randn(t, h, d, generator=g).to(dt).to(gpu) for h in (hq, hkv))
    pos = torch.randint(0, 1 << 20, (t,), generator=g).to(torch.int32).to(gpu)
    pos[0] = (1 << 31) - 1  # the furthest
    pos[-1] = 0
    for transposed in (False, True):
        qo, ko = cev_hip.rope(q, k, pos, rot, interleaved=interleaved, transposed=transposed)
        for x, y in ((q, qo), (k, ko)):
            want, size = _rope_oracle(x, pos, rot, interleaved, transposed)
            _rope_close(y, want, size, kind)
            assert torch.equal(y[..., rotary:], x[..., rotary:])
    # in place
    q2, k2 = q.clone(), k.clone()
    cev_hip.rope(q2, k2, pos, rot, interleaved=interleaved, q_out=q2, k_out=k2, transposed=True)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("page,t", [(1, 9), (16, 1), (16, 75), (64, 300)])
def test_rope_stores_into_pages(gpu, kind, page, t):
    """Strided inputs, caches of either head order, slots that store nothing, everything else left as it was."""
    import torch
    g = torch.Generator().manual_seed(page + t)
    dt = _torch_type(kind)
    hq, hkv, d = 4, 2, 128
    qkv = torch.randn(t, (hq + 2 * hkv) * d + 16, generator=g).to(dt).to(gpu)
    q, k, v = (qkv[:, a * d: b * d].view(t, b - a, d) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    n = -(-t // page) + 2
    slots = torch.randperm(n * page, generator=g)[:t].to(torch.int32)
    slots[t // 2] = -1
    slots[t // 3] = n * page
    stored = (slots >= 0) & (slots < n * page)
    rot = cev_hip.RotaryAngles(1e4, 64, gpu)
    pos = torch.randint(0, 5000, (t,), generator=g).to(torch.int32).to(gpu)
    kc = torch.full((n, page, hkv, d), 7.0, dtype=dt, device=gpu)
    vc = torch.full((n, hkv, page, d), 7.0, dtype=dt, device=gpu).transpose(1, 2)
    qo, ko, vo = cev_hip.rope(q, k, pos, rot, v_in=v, k_out=kc, v_out=vc, slots=slots.to(gpu))
    assert ko is kc and vo is vc
    want, size = _rope_oracle(q, pos, rot, False, False)
    _rope_close(qo, want, size, kind)
    want, size = _rope_oracle(k, pos, rot, False, False)
    at = slots[stored].long()
    rows = lambda c: c.reshape(n * page, hkv, d).cpu()  # noqa: E731
    _rope_close(rows(kc)[at], want[stored], size[stored], kind)
    assert torch.equal(rows(vc)[at], v.cpu()[stored])
    rest = torch.ones(n * page, dtype=torch.bool)
    rest[at] = False
    assert (rows(kc)[rest] == 7).all() and (rows(vc)[rest] == 7).all()
    # without v
    kc2 = torch.full_like(kc, 7.0)
    cev_hip.rope(q, k, pos, rot, k_out=kc2, slots=slots.to(gpu))
    assert torch.equal(kc, kc2)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_gradient(gpu, interleaved):
    """transposed=True is the gradient: <g, rope(x)> = <rope^T(g), x>, and the
    difference quotient of the (linear) map."""
    import torch
    g = torch.Generator().manual_seed(5)
    t, h, d, rotary = 9, 3, 128, 96
    rot = cev_hip.RotaryAngles(1e6, rotary, gpu, scaling="yarn", factor=8.0, original=4096)
    x, dy = (torch.randn(t, h, d, generator=g).to(gpu) for _ in range(2))
    pos = torch.randint(0, 1 << 20, (t,), generator=g).to(torch.int32).to(gpu)
    f = lambda a, tr: cev_hip.rope(a, a, pos, rot, interleaved=interleaved, transposed=tr)[0]  # noqa: E731
    dx = f(dy, True)
    # 2^-21 of a pair's size each, over t h d products of two such rows
    total = float((x.double().norm() * dy.double().norm())) * rot.factor
    assert abs(float((dy.double() * f(x, False).double()).sum() - (dx.double() * x.double()).sum())) <= 2.0 ** -20 * total
    e = torch.zeros_like(x)
    for i in (0, 1, 47, 48, 95, 96, 127):
        e.zero_()
        e[4, 1, i] = 1.0
        quotient = float((dy.double() * (f(x + e, False).double() - f(x - e, False).double())).sum() / 2)
        size = float((x.abs().max() + 1) * dy.abs().max()) * rot.factor
        assert abs(quotient - float(dx[4, 1, i])) <= 2.0 ** -18 * size


# ---------------------------------------------------------------------------
# Attention over pages


class _Paged:
    """Requests of `past` cached and `new` new tokens over shuffled pages."""

    def __init__(self, dev, past, new, hq, hkv, d, kind, page, seed=0, pad=0, head_major=False, spare=3, fill=None):
        import torch
        g = torch.Generator().manual_seed(seed)
        dt = _torch_type(kind)
        self.past, self.new, self.page, self.kind = list(past), list(new), page, kind
        total = [p + n for p, n in zip(past, new)]
        pages = [-(-x // page) for x in total]
        self.n_pages = sum(pages) + spare
        self.max_pages = max(1, max(pages)) + 1
        order = torch.randperm(self.n_pages, generator=g).tolist()
        table, at = [], 0
        for x in pages:
            table.append(order[at: at + x] + [-1] * (self.max_pages - x))
            at += x
        self.t = max(1, sum(new)) + pad
        shape = (self.n_pages, hkv, page, d) if head_major else (self.n_pages, page, hkv, d)
        order_of = (lambda x: x.transpose(1, 2)) if head_major else (lambda x: x)
        self.k, self.v = (order_of(torch.randn(*shape, generator=g).to(dt).to(dev)) for _ in range(2))
        self.q = torch.randn(self.t, hq, d, generator=g).to(dt).to(dev)
        self.table = torch.tensor(table, dtype=torch.int32, device=dev)
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=dev)
        self.lengths = torch.tensor(total, dtype=torch.int32, device=dev)
        self.hq, self.hkv, self.d = hq, hkv, d

    def keys(self, r, cache):
        """(keys, hkv, d) of request r in 64 bits."""
        n = self.past[r] + self.new[r]
        rows = self.table[r, : -(-n // self.page)].long()
        return cache[rows].flatten(0, 1)[:n].double()

    def attention(self, **kw):
        return cev_hip.PagedAttention(self.q, self.k, self.table, **kw)

    def run(self, out=None, stream=None, **kw):
        import torch
        att = self.attention(**kw)
        out = torch.full_like(self.q, 5.0) if out is None else out
        att.plan(self.cu, self.lengths, stream=stream)
        att(self.q, self.k, self.v, self.table, out=out, stream=stream)
        return out

    def exact(self, r, window=0, sinks=0, scale=None, **_):
        """(rows, hq, d) of request r, and the size that its errors are measured by: sum of p |v| and the largest |score|."""
        import torch
        k, v = self.keys(r, self.k), self.keys(r, self.v)
        r0 = sum(self.new[:r])
        q = self.q[r0: r0 + self.new[r]].double()
        g = self.hq // self.hkv
        kk, vv = (x.repeat_interleave(g, 1) for x in (k, v))
        s = torch.einsum("qhd,khd->hqk", q.cpu(), kk.cpu()) * (1 / math.sqrt(self.d) if scale is None else scale)
        p = torch.arange(self.past[r], self.past[r] + self.new[r])[:, None]
        j = torch.arange(self.past[r] + self.new[r])
        seen = j <= p
        if window:
            seen &= (j > p - window) | (j < sinks)
        s = s.masked_fill(~seen, -math.inf)
        w = torch.softmax(s, -1)
        vv = vv.cpu()
        clean = torch.where(torch.isfinite(vv), vv, torch.zeros(()).double())
        o = torch.einsum("hqk,khd->qhd", w, clean)
        size = torch.einsum("hqk,khd->qhd", w, clean.abs())
        big = float(s[torch.isfinite(s)].abs().max())
        return o, size, big

    def check(self, out, what="", **kw):
        import torch
        out = out.cpu()
        at = 0
        for r, n in enumerate(self.new):
            if n:
                o, size, big = self.exact(r, **kw)
                # A weight's relative error: its score is a sum of d products in
                # f32, off by 2^-22 of |q||k| scale, here at most 2^-20 of the
                # largest score and of one (times the exponential's own 2^-21);
                # bf16 also rounds it to half a step, on both sides of the
                # division.  Then the output's own rounding.
                half = HALF[self.kind]
                weight = 2.0 ** -19 * (1 + big) + (2 * half if self.kind == "bf16" else 0.0)
                err = (out[at: at + n].double() - o).abs()
                bound = weight * size + half * o.abs() * 1.01 + 1e-30
                worst = float((err / bound).max())
                assert worst <= 1, (what, r, worst, float(err.max()))
            at += n
        assert bool((out[at:] == 5.0).all()), "rows of no request"


SHAPES = [("bf16", 8, 2, 128), ("bf16", 4, 4, 128), ("bf16", 4, 2, 256), ("bf16", 16, 2, 128), ("f32", 4, 2, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,hq,hkv,d", SHAPES)
@pytest.mark.parametrize("past,new,page", [
    ([0], [1], 16), ([0, 0, 5], [1, 2, 1], 16), ([31, 32, 33, 15, 16, 63], [1] * 6, 16), ([300], [1], 32),
    ([0, 7, 100], [37, 0, 5], 16), ([129, 1000, 0], [3, 70, 130], 64), ([2047], [9], 1024), ([500] * 3, [1, 8, 40], 128)])
def test_attention_over_pages(gpu, kind, hq, hkv, d, past, new, page):
    p = _Paged(gpu, past, new, hq, hkv, d, kind, page, seed=len(past) + page, pad=2)
    p.check(p.run())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,hq,hkv,d", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (32, 0), (33, 4), (100, 64), (64, 200), (5000, 10)])
def test_attention_with_a_window(gpu, kind, hq, hkv, d, window, sinks):
    """Pages that no row sees are gone: their entries point outside, their
    places hold NaN."""
    import torch
    past, new = [0, 130, 700, 33, 1000], [50, 1, 40, 2, 1]
    p = _Paged(gpu, past, new, hq, hkv, d, kind, 16, seed=window + sinks, pad=1, head_major=True)
    for r in range(len(past)):
        lo = past[r] - window + 1  # keys below are seen by no row, but for the first ones
        for j in range(p.max_pages):
            if j * 16 >= sinks and (j + 1) * 16 <= lo:
                page = int(p.table[r, j])
                p.k[page], p.v[page] = math.nan, math.nan
                p.table[r, j] = [-1, 10 ** 9, page][j % 3]
    out = p.run(window=window, sinks=sinks)
    # the oracle reads them as zeros of weight zero
    p.k, p.v = torch.nan_to_num(p.k), torch.nan_to_num(p.v)
    p.table.clamp_(0, p.n_pages - 1)
    p.check(out, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,hq,hkv,d", SHAPES)
def test_attention_long_keys_split(gpu, kind, hq, hkv, d):
    """One request's keys over many workgroups, twice with one plan, the same bits each time."""
    import torch
    p = _Paged(gpu, [20011], [1], hq, hkv, d, kind, 16, seed=9)
    att = p.attention()
    att.plan(p.cu, p.lengths)
    a = att(p.q, p.k, p.v, p.table)
    b = att(p.q, p.k, p.v, p.table)
    p.check(a)
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,hq,hkv,d", SHAPES)
def test_attention_of_a_long_prompt(gpu, kind, hq, hkv, d):
    p = _Paged(gpu, [600, 0], [420, 777], hq, hkv, d, kind, 32, seed=4, pad=3)
    p.check(p.run())
    p.check(p.run(window=100, sinks=4), window=100, sinks=4)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,d", [("bf16", 128), ("bf16", 256), ("f32", 128)])
@pytest.mark.parametrize("requests,past_hi,new_hi", [(40, 700, 1), (70, 300, 9), (9, 1500, 200), (200, 40, 3), (3, 60, 900), (33, 2500, 2)])
def test_attention_of_more_work_than_workgroups(gpu, kind, d, requests, past_hi, new_hi):
    """Sixteen KV heads leave 16 or 32 workgroups a head: tiles in rounds, cut
    ones, shared-out ones.  Twice with one plan: the same bits."""
    import torch
    rng = random.Random(requests)
    past = [rng.choice([0, rng.randint(0, past_hi), past_hi]) for _ in range(requests)]
    new = [rng.choice([1, new_hi, rng.randint(0, new_hi)]) for _ in range(requests)]
    p = _Paged(gpu, past, new, 16, 16, d, kind, 16, seed=requests)
    for kw in ({}, dict(window=50, sinks=5)):
        att = p.attention(**kw)
        att.plan(p.cu, p.lengths)
        out = att(p.q, p.k, p.v, p.table, out=torch.full_like(p.q, 5.0))
        p.check(out, **kw)
        assert torch.equal(att(p.q, p.k, p.v, p.table, out=torch.full_like(p.q, 5.0)), out)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,hq,hkv,d", SHAPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", ["k", "v"])
def test_values_that_a_row_does_not_see_do_not_reach_it(gpu, kind, hq, hkv, d, value, which):
    """An infinity or NaN at one new token: the rows before it are clean, it
    and the rows after it are as the definition says; with a window also the
    rows that have left it behind."""
    import torch
    past, new, at = [70], [90], 70 + 41
    for kw in ({}, dict(window=20, sinks=2)):
        p = _Paged(gpu, past, new, hq, hkv, d, kind, 16, seed=11)
        clean = p.run(**kw)
        _, size, big = p.exact(0, **kw)
        # f32 rows that share a workgroup with a row that is not finite are summed
        # again on the f32 unit: both sums are within the bound of _Paged.check
        slack = 2.0 ** -18 * (1 + big) * size if kind == "f32" else torch.zeros_like(size)
        same = lambda a, b, rows, heads, cols: bool(  # noqa: E731
            ((a - b).double().cpu().abs() <= slack)[rows][:, heads][..., cols].all())
        cache = getattr(p, which)
        page, off = int(p.table[0, at // 16]), at % 16
        if which == "v":
            cache[page, off, 0, 5] = value
        else:
            cache[page, off, 0] = value
        out = p.run(**kw)
        g = hq // hkv
        sees = torch.zeros(90, dtype=torch.bool)
        sees[41: 41 + kw.get("window", 90)] = True
        every = torch.ones(d, dtype=torch.bool)
        assert same(out, clean, ~sees, slice(None), every)
        assert same(out, clean, slice(None), slice(g, None), every)  # the other heads' keys
        rows = out[sees.to(gpu), :g]
        if which == "v":
            col = rows[..., 5].float()
            assert bool((col.isnan() if math.isnan(value) else col == value).all())
            assert same(out, clean, sees, slice(0, g), torch.arange(d) != 5)
        elif math.isnan(value):
            assert bool(rows.isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,d", [("bf16", 128), ("bf16", 256), ("f32", 128)])
@pytest.mark.parametrize("requests,past_hi,new_hi", [(513, 90, 2), (700, 40, 1), (4096, 20, 2)])
def test_attention_of_many_requests(gpu, kind, d, requests, past_hi, new_hi):
    rng = random.Random(requests)
    past = [rng.randint(0, past_hi) for _ in range(requests)]
    p = _Paged(gpu, past, [rng.randint(0, new_hi) for _ in range(requests)], 2, 1, d, kind, 16, seed=requests, pad=1)
    p.check(p.run())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,hq,hkv,d", [("bf16", 6, 3, 128), ("bf16", 40, 5, 128), ("bf16", 300, 300, 128), ("bf16", 14, 7, 256), ("f32", 3, 3, 128),
                                           ("bf16", 1, 1, 128)])
def test_attention_of_odd_head_counts(gpu, kind, hq, hkv, d):
    """KV heads that do not divide the workgroups, and more heads than those."""
    p = _Paged(gpu, [0, 200, 33], [40, 1, 9], hq, hkv, d, kind, 16, seed=hkv, pad=2)
    for kw in ({}, dict(window=2 ** 31 - 1), dict(window=30, sinks=2 ** 31 - 1)):
        p.check(p.run(**kw), kw, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,d,many", [("bf16", 128, False), ("bf16", 128, True), ("bf16", 256, False), ("bf16", 256, True), ("f32", 128, False)])
def test_attention_in_place_of_q(gpu, kind, d, many):
    import torch
    p = (_Many if many else _Paged)(gpu, [0, 3000, 33], [40, 70, 1], 8, 2, d, kind, 16, seed=2)
    want = p.run()
    assert torch.equal(p.run(out=p.q), want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,hq,hkv,d", [("bf16", 8, 2, 128), ("bf16", 4, 2, 256), ("f32", 4, 2, 128)])
def test_requests_that_share_pages(gpu, kind, hq, hkv, d):
    """A common beginning lies in the same pages, and one page is twice in a request's table."""
    p = _Paged(gpu, [100, 130, 64], [3, 1, 20], hq, hkv, d, kind, 16, seed=4)
    p.table[1, :6] = p.table[0, :6]
    p.table[2, 3] = p.table[2, 1]
    p.check(p.run())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_two_graphs_of_one_object(gpu, kind):
    """A graph of a decoding step and one of a chunk's, of the same work buffer,
    replayed in turn, with eager calls and other lengths between."""
    import torch
    p = _Paged(gpu, [700, 40, 2000], [1, 33, 5], 8, 2, 128, kind, 16, seed=13, pad=3)
    att, out = p.attention(), torch.empty_like(p.q)
    att.plan(p.cu, p.lengths)(p.q, p.k, p.v, p.table, out=out)
    torch.cuda.synchronize()
    steps = ([700, 40, 2000], [1, 33, 5]), ([701, 0, 1998], [1, 1, 7])
    graphs = []
    sets = [tuple(torch.tensor(x, dtype=torch.int32, device=gpu) for x in (np.concatenate([[0], np.cumsum(new)]), np.add(past, new))) for past, new in steps]
    for cu, lengths in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            att.plan(cu, lengths)
            att(p.q, p.k, p.v, p.table, out=out)
    for i in (0, 1, 1, 0, 2, 1, 0):
        out.fill_(5.0)
        if i == 2:
            att.plan(*sets[0])(p.q, p.k, p.v, p.table, out=out)
            i = 0
        else:
            graphs[i].replay()
        torch.cuda.synchronize()
        p.past, p.new = steps[i]
        p.check(out, i)


@pytest.mark.gpu
def test_tables_and_rope_on_another_stream(gpu):
    import torch
    s = torch.cuda.Stream()
    a, b = (_Tables(gpu, [5, 40, 0, 17], 16, 8, 9, seed=3, max_tokens=20) for _ in range(2))
    new = [3, -1, 8, 1]
    torch.cuda.synchronize()
    want = a.expect(new)
    a.step(new)
    b.step(new, stream=s)
    a.check(want)
    b.check(want)
    rot = cev_hip.RotaryAngles(1e6, 128, gpu)
    q, k = torch.randn(20, 4, 128, device=gpu), torch.randn(20, 2, 128, device=gpu)
    here = cev_hip.rope(q, k, a.pos, rot)
    torch.cuda.synchronize()
    there = cev_hip.rope(q, k, a.pos, rot, stream=s)
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(here, there))


class _Many(_Paged):
    """The same, with one more request behind them of so many rows that the plan
    sends all requests of more than 32 query slots to the kernel of many rows.
    Its own rows are only looked at for being finite."""

    def __init__(self, dev, past, new, hq, hkv, d, kind, page, window=0, **kw):
        rows, work = 32 * hkv // hq, 32 * (512 // hkv) if d == 128 else 96 * (256 // hkv)
        each = (window + rows + 30) // 32 if window else 64  # sub-tiles that a tile sees at least
        super().__init__(dev, [*past, window or 2048], [*new, rows * (work // each + 2)], hq, hkv, d, kind, page, **kw)

    def run(self, out=None, stream=None, **kw):
        import torch
        att = self.attention(**kw)
        out = torch.full_like(self.q, 5.0) if out is None else out
        att.plan(self.cu, self.lengths, stream=stream)
        assert int(att.work[12:16].view(torch.int32)) > 0  # workgroups of the second list
        return att(self.q, self.k, self.v, self.table, out=out, stream=stream)

    def check(self, out, what="", **kw):
        out, all_new = out.clone(), self.new
        rows = slice(sum(all_new[:-1]), sum(all_new))
        assert bool(out[rows].isfinite().all())
        out[rows] = 5.0
        self.new = all_new[:-1]
        super().check(out, what, **kw)
        self.new = all_new


MANY_SHAPES = [("bf16", 8, 2, 128), ("bf16", 4, 4, 128), ("bf16", 16, 2, 128), ("bf16", 4, 2, 256), ("bf16", 8, 1, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,hq,hkv,d", MANY_SHAPES)
@pytest.mark.parametrize("past,new,page,window,sinks", [
    ([0, 7, 100], [37, 0, 50], 16, 0, 0), ([0, 0, 31, 64], [33, 64, 65, 257], 16, 0, 0), ([129, 1000, 0], [70, 1, 130], 64, 0, 0),
    ([20011], [40], 1024, 0, 0), ([0, 130, 700, 33], [50, 40, 300, 2], 16, 1, 0), ([0, 130, 700], [50, 40, 70], 16, 7, 3),
    ([0, 130, 700], [50, 40, 70], 32, 33, 4), ([10, 1000], [500, 40], 16, 64, 200), ([0, 3000], [100, 100], 16, 1000, 70)])
def test_attention_of_many_rows(gpu, kind, hq, hkv, d, past, new, page, window, sinks):
    import torch
    kw = dict(window=window, sinks=sinks) if window else {}
    p = _Many(gpu, past, new, hq, hkv, d, kind, page, seed=len(past) + page, pad=2, window=window)
    out = p.run(**kw)
    p.check(out, **kw)
    assert torch.equal(p.run(**kw), out)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,hq,hkv,d", MANY_SHAPES[:4])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", ["k", "v"])
def test_values_that_one_of_many_rows_does_not_see(gpu, kind, hq, hkv, d, value, which):
    import torch
    past, new, at = [70], [90], 70 + 41
    for kw in ({}, dict(window=20, sinks=2)):
        p = _Many(gpu, past, new, hq, hkv, d, kind, 16, seed=11, window=kw.get("window", 0))
        clean = p.run(**kw)[:90]
        cache = getattr(p, which)
        page, off = int(p.table[0, at // 16]), at % 16
        if which == "v":
            cache[page, off, 0, 5] = value
        else:
            cache[page, off, 0] = value
        out = p.run(**kw)[:90]
        g = hq // hkv
        sees = torch.zeros(90, dtype=torch.bool, device=gpu)
        sees[41: 41 + kw.get("window", 90)] = True
        assert torch.equal(out[~sees], clean[~sees]) and torch.equal(out[:, g:], clean[:, g:])
        rows = out[sees][:, :g]
        if which == "v":
            col = rows[..., 5].float()
            assert bool((col.isnan() if math.isnan(value) else col == value).all())
            assert torch.equal(rows[..., torch.arange(d) != 5], clean[sees][:, :g][..., torch.arange(d) != 5])
        elif math.isnan(value):
            assert bool(rows.isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("d", [128, 256])
def test_bad_pages_of_many_rows(gpu, d):
    """A page outside the cache that only the later rows of a request see, and one in a request of its own."""
    p = _Many(gpu, [20, 100], [60, 70], 8, 2, d, "bf16", 16)
    want = p.run()
    p.table[0, 4], p.table[1, 0] = p.n_pages, -1
    out = p.run()
    assert bool(out[60:130].isnan().all()) and bool(out[44:60].isnan().all())
    assert bool((out[130:] == want[130:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("d", [128, 256])
def test_many_rows_strides_and_far_pages(gpu, d):
    """Caches with strides of their own whose pages lie more than 4 GiB in, rows
    inside larger buffers, an odd block table stride, another stream."""
    import torch
    p = _Many(gpu, [40, 333, 0], [50, 33, 200], 8, 2, d, "bf16", 16, seed=6)
    want = p.run()
    n_pages = (5 << 30) // (2 * 16 * 2 * (d + 16))
    far = torch.arange(p.n_pages, device=gpu) * (n_pages // p.n_pages - 1) + 5
    for name in ("k", "v"):
        wide = torch.empty(n_pages, 16, 2, d + 16, dtype=torch.bfloat16, device=gpu)[..., :d]
        wide[far] = getattr(p, name)
        setattr(p, name, wide)
    p.n_pages = n_pages
    moved = torch.where(p.table >= 0, far[p.table.clamp(min=0).long()], -1).to(torch.int32)
    p.table = torch.full((moved.shape[0], p.max_pages + 3), -1, dtype=torch.int32, device=gpu)[:, : p.max_pages]
    p.table.copy_(moved)
    q = torch.zeros(p.t, 8, d + 8, dtype=torch.bfloat16, device=gpu)[..., :d]
    q.copy_(p.q)
    p.q = q
    out = torch.full((p.t, 16, d), 5.0, dtype=torch.bfloat16, device=gpu)[:, ::2]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    p.run(out=out, stream=s)
    s.synchronize()
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("order", ["up", "down", "one"])
def test_large_scores_of_many_rows(gpu, d, order):
    """The running maximum moves, stays, or sits at one key."""
    import torch
    p = _Many(gpu, [800], [103], 4, 2, d, "bf16", 16, seed=3)
    place = torch.zeros(p.n_pages, 16, device=gpu)
    for i, page in enumerate(p.table[0, : -(-903 // 16)].tolist()):
        place[page] = torch.arange(16, device=gpu) + 16 * i
    size = {"up": place / 903, "down": 1 - place / 903, "one": (place == 450).float()}[order]
    p.q.copy_(p.q.sign())
    p.k.copy_((size[..., None, None] * 25 * p.q[0, 0].float()).to(p.k.dtype).expand_as(p.k))
    p.check(p.run(), order)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_attention_of_large_scores(gpu, kind):
    """Scores of several hundred that rise with the key, fall, or sit at one key: the running maximum moves or stays."""
    import torch
    for order in ("up", "down", "one"):
        p = _Paged(gpu, [900], [3], 4, 2, 128, kind, 16, seed=3)
        j = torch.arange(p.n_pages * 16, device=gpu).view(p.n_pages, 16)
        place = torch.zeros(p.n_pages, 16, device=gpu)
        for i, page in enumerate(p.table[0, : -(-903 // 16)].tolist()):
            place[page] = torch.arange(16, device=gpu) + 16 * i
        size = {"up": place / 903, "down": 1 - place / 903, "one": (place == 450).float()}[order]
        p.q.copy_(p.q.sign())
        p.k.copy_((size[..., None, None] * 25 * p.q[0, 0].float()).to(p.k.dtype).expand_as(p.k))
        assert j.numel()
        p.check(p.run(), order)


@pytest.mark.gpu
def test_lengths_and_pages_out_of_bounds_give_nan(gpu):
    import torch
    p = _Paged(gpu, [20, 30], [3, 4], 4, 2, 128, "bf16", 16, pad=2)
    for name, value in (("cu", [0, 3, 99]), ("cu", [0, 5, 3]), ("cu", [-1, 3, 7]), ("cu", [0, 2 ** 31 - 1, 7]), ("lengths", [2, 34]),
                        ("lengths", [23, 10 ** 9]), ("lengths", [23, -5])):
        old = getattr(p, name).clone()
        getattr(p, name).copy_(torch.tensor(value, dtype=torch.int32))
        assert bool(p.run().isnan().all()), (name, value)
        getattr(p, name).copy_(old)
    assert bool(p.run(max_new=3).isnan().all())  # request 1 has four
    # one request's page
    p.table[1, 1] = p.n_pages
    out = p.run()
    assert bool(out[3:7].isnan().all()) and not out[:3].isnan().any() and bool((out[7:] == 5).all())
    # no plan yet, another descriptor's plan
    att = p.attention()
    assert bool(att(p.q, p.k, p.v, p.table).isnan().all())
    other = p.attention(window=8)
    other.plan(p.cu, p.lengths)
    att.work.copy_(other.work[: att.work.numel()])
    assert bool(att(p.q, p.k, p.v, p.table).isnan().all())
    # no rows at all
    p.cu.zero_()
    assert bool((p.run() == 5).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_attention_strides_and_streams(gpu, kind):
    """Rows and caches inside larger buffers, odd block table strides, another stream than the current one."""
    import torch
    p = _Paged(gpu, [40, 333], [5, 33], 8, 4, 128, kind, 16, seed=6)
    want = p.run()
    wide = lambda x, dim, by: torch.cat([x, torch.full_like(x, 9.0)], dim).narrow(dim, 0, x.shape[dim]) if by else x  # noqa: E731
    q2 = torch.zeros(p.t, 8, 136, dtype=p.q.dtype, device=gpu)[..., :128]
    q2.copy_(p.q)
    table = torch.full((2, p.max_pages + 5), -1, dtype=torch.int32, device=gpu)[:, : p.max_pages]
    table.copy_(p.table)
    p.q, p.table = q2, table
    p.k, p.v = wide(p.k, 2, 1), wide(p.v, 3, 1)
    out = torch.full((p.t, 16, 128), 5.0, dtype=q2.dtype, device=gpu)[:, ::2]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    p.run(out=out, stream=s)
    s.synchronize()
    assert torch.equal(out, want)


@pytest.mark.gpu
def test_cache_beyond_32_bit_offsets(gpu):
    """Pages that lie more than 4 GiB into the caches."""
    import torch
    page, hkv, d = 16, 2, 128
    n_pages = (9 << 30) // (2 * page * hkv * d)  # 9 GiB each
    k = torch.empty(n_pages, page, hkv, d, dtype=torch.bfloat16, device=gpu)
    v = torch.empty_like(k)
    p = _Paged(gpu, [100, 50], [2, 1], 8, hkv, d, "bf16", page, seed=8)
    far = torch.arange(p.n_pages, device=gpu) * (n_pages // p.n_pages - 1) + (n_pages - 1) % 7
    k[far], v[far] = p.k, p.v
    want = p.run()
    p.k, p.v, p.n_pages = k, v, n_pages
    p.table = torch.where(p.table >= 0, far[p.table.clamp(min=0).long()], -1).to(torch.int32)
    assert int(p.table.max()) * page * hkv * d * 2 > 1 << 32  # bytes
    assert torch.equal(p.run(), want)
    # and the stores
    rot = cev_hip.RotaryAngles(1e4, 128, gpu)
    x = torch.randn(3, hkv, d, device=gpu).bfloat16()
    slots = torch.tensor([int(far[-1]) * page + 3, 5, n_pages * page - 1], dtype=torch.int32, device=gpu)
    cev_hip.rope(x, x, torch.zeros(3, dtype=torch.int32, device=gpu), rot, v_in=x, k_out=k, v_out=v, slots=slots)
    for i, s in enumerate(slots.tolist()):
        assert torch.equal(k[s // page, s % page], x[i]) and torch.equal(v[s // page, s % page], x[i])


# ---------------------------------------------------------------------------
# Together


def _model_step(state, x, out):
    """One layer's step: bookkeeping, rotary and stores, attention."""
    s = state
    cev_hip.paged_tables(s["lengths"], s["new"], s["table"], s["page"], s["cu"], s["pos"], s["slots"], free=s["free"], ring=s["ring"])
    q, k, v = x
    qr, _, _ = cev_hip.rope(q, k, s["pos"], s["rot"], v_in=v, q_out=s["q"], k_out=s["k"], v_out=s["v"], slots=s["slots"])
    s["att"].plan(s["cu"], s["lengths"])
    s["att"](qr, s["k"], s["v"], s["table"], out=out)


def _serving(gpu, requests=3, page=16, room=48, kind="bf16", window=0, sinks=0, max_pages=12):
    import torch
    hq, hkv, d = 4, 2, 128
    dt = _torch_type(kind)
    n_pages = requests * max_pages
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=gpu)  # noqa: E731
    s = dict(lengths=i(requests), new=i(requests), table=torch.full((requests, max_pages), -1, dtype=torch.int32, device=gpu), page=page,
             cu=i(requests + 1), pos=i(room), slots=i(room), rot=cev_hip.RotaryAngles(1e6, d, gpu))
    s["free"], s["ring"] = cev_hip.free_ring(n_pages, gpu)
    # pages that nobody has written hold NaN
    s["k"], s["v"] = (torch.full((n_pages, page, hkv, d), math.nan, dtype=dt, device=gpu) for _ in range(2))
    s["q"] = torch.zeros(room, hq, d, dtype=dt, device=gpu)
    s["att"] = cev_hip.PagedAttention(s["q"], s["k"], s["table"], window=window, sinks=sinks)
    return s, (hq, hkv, d)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("captured", [False, True])
def test_a_run_of_steps(gpu, kind, window, sinks, captured):
    """Prompts, single tokens, a request that ends and another in its place:
    every step's rows against attention over each request's whole history.
    Captured, one graph is replayed for every step."""
    import torch
    s, (hq, hkv, d) = _serving(gpu, kind=kind, window=window, sinks=sinks)
    room = s["q"].shape[0]
    g = torch.Generator().manual_seed(1)
    dt = s["q"].dtype
    x = [torch.zeros(room, h, d, dtype=dt, device=gpu) for h in (hq, hkv, hkv)]
    out = torch.zeros_like(s["q"])
    graph = None
    if captured:
        _model_step(s, x, out)  # nothing is new: no row
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _model_step(s, x, out)
    history = [[] for _ in range(3)]  # (k, v) rows after rotary, as stored
    steps = [(20, 3, 0), (1, 17, 30), (1, 1, 1), (1, -1, 1), (16, 5, 0), (1, 1, 1), (1, 33, 1), (-1, 1, -1), (2, 1, 40)]
    for n_step, new in enumerate(steps):
        rows = [torch.randn(room, h, d, generator=g).to(dt).to(gpu) for h in (hq, hkv, hkv)]
        for a, b in zip(x, rows):
            a.copy_(b)
        s["new"].copy_(torch.tensor(new, dtype=torch.int32))
        out.fill_(5.0)
        if graph:
            graph.replay()
        else:
            _model_step(s, x, out)
        torch.cuda.synchronize()
        assert s["ring"].tolist()[2:] == [0, 0]
        at = 0
        for r, n in enumerate(new):
            if n < 0:
                history[r] = []
                continue
            pos = torch.arange(len(history[r]), len(history[r]) + n)
            if not n:
                continue
            qr, _ = _rope_oracle(rows[0][at: at + n], pos, s["rot"], False, False)
            kr, _ = _rope_oracle(rows[1][at: at + n], pos, s["rot"], False, False)
            history[r] += [(a, b) for a, b in zip(kr.to(dt), rows[2][at: at + n].cpu())]
            k = torch.stack([a for a, _ in history[r]]).double().repeat_interleave(hq // hkv, 1)
            v = torch.stack([b for _, b in history[r]]).double().repeat_interleave(hq // hkv, 1)
            score = torch.einsum("qhd,khd->hqk", qr.to(dt).double(), k) / math.sqrt(d)
            j = torch.arange(len(history[r]))
            seen = j <= pos[:, None]
            if window:
                seen &= (j > pos[:, None] - window) | (j < sinks)
            w = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
            o, size = torch.einsum("hqk,khd->qhd", w, v), torch.einsum("hqk,khd->qhd", w, v.abs())
            # as in _Paged.check; a rotated q or k may also be rounded to the
            # other side (one step of each value), which moves a score by at
            # most 4 half steps of |q||k| scale, so each weight by twice that
            qk = float((qr.norm(dim=-1).max() * k.norm(dim=-1).max()) / math.sqrt(d))
            half = HALF[kind]
            bound = (2.0 ** -19 * (1 + qk) + (2 * half if kind == "bf16" else 0) + 8 * half * qk) * size + half * o.abs() * 1.01
            err = (out[at: at + n].double().cpu() - o).abs()
            assert bool((err <= bound).all()), (n_step, r, float((err / bound).max()))
            at += n
        assert bool((out[at:] == 5.0).all())
    held = sum(-(-int(n) // s["page"]) for n in s["lengths"].tolist())
    assert s["ring"].tolist()[1] + held == s["free"].shape[0]
    taken = [e for r, n in zip(s["table"].tolist(), s["lengths"].tolist()) for e in r[: -(-n // s["page"])]]
    head, count = s["ring"].tolist()[:2]
    free = [s["free"].tolist()[(head + i) % len(s["free"])] for i in range(count)]
    assert sorted(taken + free) == list(range(len(s["free"])))


@pytest.mark.gpu
def test_a_failed_step_leaves_the_caches(gpu):
    """Too few pages: no row is stored or attended, and the next step goes on."""
    import torch
    s, (hq, hkv, d) = _serving(gpu, max_pages=2)
    x = [torch.randn(48, h, d, device=gpu).bfloat16() for h in (hq, hkv, hkv)]
    out = torch.full_like(s["q"], 5.0)
    s["ring"][1] = 1
    s["new"].copy_(torch.tensor([10, 20, 1], dtype=torch.int32))
    _model_step(s, x, out)
    assert s["ring"].tolist() == [0, 1, 4, 0] and bool((out == 5).all()) and bool(s["k"].isnan().all())
    s["new"].copy_(torch.tensor([10, 0, 0], dtype=torch.int32))
    _model_step(s, x, out)
    assert s["ring"].tolist() == [1, 0, 0, 0] and not out[:10].isnan().any() and bool((out[10:] == 5).all())


@pytest.mark.gpu
def test_the_caches_serve_the_fused_norm_and_rope(gpu):
    """qknorm_rope_kv stores into the same pages, as their slots."""
    import torch
    s, (hq, hkv, d) = _serving(gpu, kind="bf16")
    s["new"].copy_(torch.tensor([9, 0, 20], dtype=torch.int32))
    cev_hip.paged_tables(s["lengths"], s["new"], s["table"], s["page"], s["cu"], s["pos"], s["slots"], free=s["free"], ring=s["ring"])
    x = [torch.randn(48, h, d, device=gpu).bfloat16() for h in (hq, hkv, hkv)]
    w = torch.ones(d, device=gpu).bfloat16()
    rot = cev_hip.Rotary(1e6, d, 64, torch.bfloat16, gpu)
    slots_view = lambda c: c.view(-1, hkv, d)  # noqa: E731
    cev_hip.qknorm_rope_kv(*x, w, w, s["pos"], rot, 1e-6, s["q"], slots_view(s["k"]), slots_view(s["v"]), slots=s["slots"],
                           n_slots=s["free"].shape[0] * s["page"])
    kept = s["slots"].tolist()
    dense = torch.zeros(48, hkv, d, device=gpu).bfloat16()
    cev_hip.qknorm_rope(x[0], x[1], w, w, s["pos"], rot, 1e-6, k_out=dense)
    for i in range(29):
        assert torch.equal(slots_view(s["k"])[kept[i]], dense[i]) and torch.equal(slots_view(s["v"])[kept[i]], x[2][i])
    s["att"].plan(s["cu"], s["lengths"])
    out = s["att"](s["q"], s["k"], s["v"], s["table"])
    assert not out[:29].isnan().any()


@pytest.mark.gpu
def test_steps_on_two_streams(gpu):
    """Two caches' steps at once, each on its own stream with its own objects."""
    import torch
    sides = []
    for i in range(2):
        s, (hq, hkv, d) = _serving(gpu, max_pages=40)
        x = [torch.randn(48, h, d, generator=torch.Generator().manual_seed(i)).bfloat16().to(gpu) for h in (hq, hkv, hkv)]
        s["new"].copy_(torch.tensor([16, 1, 12 + i], dtype=torch.int32))
        sides.append((s, x, torch.full_like(s["q"], 5.0), torch.cuda.Stream()))
    alone = []
    for i in range(2):
        s, x, out, _ = sides[i]
        keep = {k: s[k].clone() for k in ("lengths", "table", "free", "ring", "k", "v")}
        for _ in range(5):
            _model_step(s, x, out)
        alone.append(out.clone())
        for k, v in keep.items():
            s[k].copy_(v)
    torch.cuda.synchronize()
    for _ in range(5):
        for s, x, out, stream in sides:
            with torch.cuda.stream(stream):
                _model_step(s, x, out)
    torch.cuda.synchronize()
    for (_, _, out, _), want in zip(sides, alone):
        assert torch.equal(out, want)


# ---------------------------------------------------------------------------
# What an ended request holds


@pytest.mark.gpu
@pytest.mark.parametrize("requests,max_pages,page,tokens", [(5, 7, 16, 40), (90, 70, 16, 300), (700, 33, 4, 5000), (70, 300, 16, 80), (3, 700, 1, 9)])
def test_an_ended_request_gives_back_what_its_row_names(gpu, requests, max_pages, page, tokens):
    """Entries that are no pages (shared ones, those given back behind a
    window) are passed over: the ring gets the others in their order, counts
    those, and never hands a page to two requests."""
    rng = random.Random(requests)
    lengths = [rng.randint(0, max_pages * page) for _ in range(requests)]
    s = _Tables(gpu, lengths, page, max_pages, spare=requests + 3, seed=requests, max_tokens=tokens, extra_stride=1)
    held = [-(-n // page) for n in lengths]
    bad = [-1, s.n_pages, 2 ** 31 - 1, -(2 ** 31)]
    for r, h in enumerate(held):
        gone = range(h) if rng.random() < 0.2 else range(0) if rng.random() < 0.2 else [j for j in range(h) if rng.random() < 0.5]
        for j in gone:
            s.table_np[r][j] = rng.choice(bad)
    s.table.copy_(s.t(s.table_np))
    new = [rng.choice([-1, -1, 0, 0]) if r else -1 for r in range(requests)]
    given = [e for r, a in enumerate(new) if a < 0 for e in s.table_np[r][: held[r]] if 0 <= e < s.n_pages]
    head, count = s.ring_np[:2]
    ring = list(s.free_np)
    for i, e in enumerate(given):
        ring[(head + count + i) % s.n_pages] = e
    table = [list(r) for r in s.table_np]
    s.step(new)
    assert s.ring.tolist() == [head, count + len(given), 0, 0] and s.free.tolist() == ring and s.table.tolist() == table
    assert s.lengths.tolist() == [0 if a < 0 else n for a, n in zip(new, lengths)]
    # whoever comes next gets pages that nobody holds
    rows = [a < 0 for a in new]
    new = [min(page * 2, tokens // requests + 1) if gone else 0 for gone in rows]
    while sum(new) > tokens:
        new[max(r for r, a in enumerate(new) if a)] = 0
    s.step(new)
    assert s.ring.tolist()[2] == 0 and min(s.slots.tolist()[: sum(new)]) >= 0
    names = [e for r in range(requests) for e in s.table.tolist()[r][: -(-s.lengths.tolist()[r] // page)] if 0 <= e < s.n_pages]
    assert len(set(names)) == len(names)
    assert not set(names) & {s.free.tolist()[(s.ring.tolist()[0] + i) % s.n_pages] for i in range(s.ring.tolist()[1])}


@pytest.mark.gpu
def test_requests_that_shared_a_prefix_end(gpu):
    """The first one holds the common pages; the others name them no more when they end."""
    s = _Tables(gpu, [40, 0, 0], 16, 4, 9, seed=5, max_tokens=60)
    common = s.table_np[0][:2]
    for r in (1, 2):  # 32 tokens of the first one's
        s.table[r, :2] = s.table[0, :2]
        s.lengths[r] = 32
    s.step([1, 10, 20])
    assert s.ring.tolist()[2] == 0
    s.table[1:, :2] = -1
    s.step([0, -1, -1])
    assert s.ring.tolist()[1:3] == [s.n_pages - 3, 0]
    s.step([-1, 0, 0])
    head, count, status, _ = s.ring.tolist()
    assert (count, status) == (s.n_pages, 0) and sorted(s.free.tolist()) == list(range(s.n_pages)) and set(common) <= set(s.free.tolist())


@pytest.mark.gpu
def test_more_pages_given_back_than_the_ring_has_room_for(gpu):
    """Counted without the entries that are no pages: with them the step would be refused."""
    s = _Tables(gpu, [64, 64], 16, 4, 0, seed=5, max_tokens=8)
    s.table_np[0][1] = s.table_np[0][3] = -1
    s.table.copy_(s.t(s.table_np))
    s.ring_np = [2, s.n_pages - 5, 0, 0]
    s.ring.copy_(s.t(s.ring_np))
    s.step([-1, -1])  # six pages, five places
    s.check(dict(status=8))
    s.ring[1] -= 1
    s.step([-1, -1])
    assert s.ring.tolist() == [2, s.n_pages, 0, 0] and s.lengths.tolist() == [0, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("requests,room", [(9, 2000), (300, 9000)])
@pytest.mark.parametrize("apart", ["both", "ring", "lengths"])
def test_tables_of_many_workgroups_write_outputs_whatever_they_held(gpu, requests, room, apart):
    """New lengths and ring state in buffers that nobody has cleared, over several steps of more than one workgroup."""
    import torch
    rng = random.Random(requests)
    s = _Tables(gpu, [rng.randint(0, 60) for _ in range(requests)], 16, 20, requests * 12, seed=3, max_tokens=room)
    for k in range(4):
        new = [rng.choice([-1, 0, 1, 20]) for _ in range(requests)]
        want = s.expect(new)
        lengths = torch.full_like(s.lengths, 77) if apart != "ring" else s.lengths
        ring = s.t([-5, 9, 3, [1, -2, 7, 2 ** 31 - 1][k]]) if apart != "lengths" else s.ring
        cev_hip.paged_tables(s.lengths, s.t(new), s.table, 16, s.cu, s.pos, s.slots, free=s.free, ring=s.ring, lengths_out=lengths, ring_out=ring)
        torch.cuda.synchronize()
        assert s.ring.tolist()[3] == 0
        s.lengths, s.ring = lengths, ring
        s.check(want, k)


def test_tables_outputs_that_cut_their_inputs_are_refused(cev):
    at = lambda a: C.c_void_p(a)  # noqa: E731
    #       requests page n_pages max_pages tokens lengths new table stride free ring lengths_out ring_out cu pos slots
    args = [8, 16, 50, 10, 0, at(4096), at(8192), at(16384), 10, at(32768), at(65536), at(69632), at(73728), at(77824), None, None, None]
    for i, where in ((11, 4096 + 4), (11, 4096 + 28), (11, 4096 - 28), (12, 65536 + 4), (12, 65536 - 12)):
        bad = list(args)
        bad[i] = at(where)
        assert _abi.lib().cev_paged_tables(*bad) == -1 and b"overlaps" in _abi.lib().cev_last_error(), (i, where)


@pytest.mark.parametrize("kw", [dict(), dict(d=256), dict(dtype=_abi.CEV_F32), dict(hq=16), dict(requests=4096)])
def test_work_size_of_the_most_tokens(cev, kw):
    """Up to 2^31 - 1 rows: the size counts the rows that the requests' pages hold, and never wraps."""
    sizes = []
    for t in (1, 9, 160, 161, 10 ** 6, 2 ** 31 - 256, 2 ** 31 - 1):
        rc, n = _work_size(_paged_desc(t=t, **kw))
        assert rc == 0
        sizes.append(n)
    # (up to t / rows + requests tiles: at t = 160 that is fewer than a tile's worth for every request)
    assert sizes == sorted(sizes) and sizes[4] == sizes[-1] < 1 << 30
    # pages for many more keys: too many tiles of them
    assert _work_size(_paged_desc(t=2 ** 31 - 1, max_pages=(2 ** 31 - 1025) // 16, n_pages=1 << 27, **kw))[0] == -2


@pytest.mark.parametrize("name,bad,says", [
    ("lengths", ("i", 3, 1), "lengths must be int32"), ("lengths", ("long", 3), "lengths must be contiguous int32 of 3"),
    ("lengths", ("i", 4), "new_len must be contiguous int32 of 4"), ("lengths", ("half", 3), "lengths must be contiguous"),
    ("new_len", ("i", 2), "new_len must be contiguous int32 of 3"), ("new_len", ("long", 3), "new_len must be contiguous"),
    ("block_table", ("i", 2, 4), r"block_table must be int32 \(3, pages\)"), ("block_table", ("i", 3, 0), "block_table must be"),
    ("block_table", ("half", 3, 4), "block_table must be"), ("block_table", ("long", 3, 4), "block_table must be"), ("block_table", ("i", 12), "block_table must be"),
    ("cu", ("i", 3), "cu must be contiguous int32 of 4"), ("cu", ("half", 4), "cu must be contiguous"), ("pos", ("half", 10), "pos must be contiguous"),
    ("pos", ("i", 10, 1), "pos must be int32"), ("pos", ("i", 9), "slots must be contiguous int32 of 9"), ("slots", ("i", 9), "slots must be contiguous int32 of 10"),
    ("slots", ("long", 10), "slots must be contiguous"), ("ring", ("i", 3), "ring must be contiguous int32 of 4"), ("ring", ("long", 4), "ring must be contiguous"),
    ("free", ("long", 20), "free must be contiguous int32 of 20"), ("free", ("half", 20), "free must be contiguous"), ("n_pages", 19, "free must be contiguous int32 of 19"),
    ("lengths_out", ("i", 4), "lengths_out must be contiguous int32 of 3"), ("ring_out", ("i", 5), "ring_out must be contiguous int32 of 4"),
    ("page_size", 1 << 40, "page_size 1099511627776 does not fit 32 bits"), ("page_size", -(1 << 31) - 1, "page_size .* does not fit"),
    ("ring", None, "ring is required"), ("free", None, "n_pages is required"), ("none", 0, "lengths must be on the GPU")])
def test_paged_tables_says_which_argument_it_refuses(cev, name, bad, says):
    """The message names the argument: a refusal for another reason (the tensors are on the CPU) is none."""
    import torch

    def tensor(kind, *shape):
        x = torch.zeros(*shape[:-1], shape[-1] * 2, dtype=torch.int64 if kind == "long" else torch.int32)
        return x[..., ::2] if kind == "half" else x[..., : shape[-1]].contiguous()
    args = dict(page_size=16)
    for k, shape in dict(lengths=(3,), new_len=(3,), block_table=(3, 4), cu=(4,), pos=(10,), slots=(10,), free=(20,), ring=(4,)).items():
        args[k] = tensor("i", *shape)
    if name != "none":
        args[name] = tensor(*bad) if isinstance(bad, tuple) else bad
    with pytest.raises(CevError, match=says) as e:
        cev.paged_tables(**args)
    assert e.value.code == -1


def test_more_pages_than_32_bits_number(cev):
    """Refused by their count, before the tensors' device is looked at."""
    import torch
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(CevError, match="n_pages 4294967296 does not fit 32 bits") as e:
        cev.paged_tables(i(3), i(3), i(3, 4), 16, i(4), i(10), i(10), ring=i(4), n_pages=1 << 32)
    assert e.value.code == -1


@pytest.mark.parametrize("change,says", [
    (dict(window=1 << 32), "window 4294967296 does not fit 32 bits"), (dict(max_new=6), "max_new 6"), (dict(max_new=0), "max_new 0"),
    (dict(max_new=(1 << 32) + 1), "max_new 4294967297 does not fit"), (dict(sinks=3), "first tokens that stay visible need a window"),
    (dict(window=-1), "window -1"), (dict(scale=0.0), "scale must be"), (dict(scale=math.inf), "scale must be"), (dict(sinks=-(1 << 40)), "sinks .* does not fit")])
def test_paged_attention_says_which_argument_it_refuses(cev, change, says):
    import torch
    with pytest.raises(CevError, match=says) as e:
        cev.PagedAttention(torch.zeros(5, 4, 128), torch.zeros(3, 16, 2, 128), torch.zeros(2, 4, dtype=torch.int32), **change)
    assert e.value.code == -1


def _rows_that_see(p, r, page, window, sinks):
    """Which of request r's new rows see a key of the page-th entry of its table."""
    rows = range(p.past[r], p.past[r] + p.new[r])
    keys = lambda at: range(page * p.page, min((page + 1) * p.page, at + 1))  # noqa: E731
    return [any(not window or j > at - window or j < sinks for j in keys(at)) for at in rows]


@pytest.mark.gpu
@pytest.mark.parametrize("many,kind,hq,hkv,d", [(False, *x) for x in SHAPES] + [(True, *x) for x in MANY_SHAPES])
@pytest.mark.parametrize("page,window,sinks", [(16, 0, 0), (16, 20, 3), (32, 40, 33), (64, 50, 0)])
def test_a_page_outside_makes_the_rows_nan_that_see_it(gpu, many, kind, hq, hkv, d, page, window, sinks):
    """Rows of the same request before such a page, and those that have left it behind their window, are as without it."""
    import torch
    kw = dict(window=window, sinks=sinks) if window else {}
    past, new = [30, 0, 200], [150, 33, 9]
    p = _Many(gpu, past, new, hq, hkv, d, kind, page, seed=8, window=window) if many else _Paged(gpu, past, new, hq, hkv, d, kind, page, seed=8)
    want = p.run(**kw)
    for r, entry, value in ((0, 5, -1), (0, 0, p.n_pages), (1, 1, 2 ** 31 - 1), (2, 0, -(2 ** 31)), (2, 200 // page, p.n_pages)):
        if entry * page >= past[r] + new[r]:
            continue
        old = int(p.table[r, entry])
        p.table[r, entry] = value
        out = p.run(**kw)
        p.table[r, entry] = old
        bad = torch.zeros(p.t, dtype=torch.bool, device=gpu)
        at = sum(new[:r])
        bad[at: at + new[r]] = torch.tensor(_rows_that_see(p, r, entry, window, sinks), device=gpu)
        assert bool(out[bad].isnan().all()), (r, entry)
        assert torch.equal(out[~bad], want[~bad]), (r, entry)
        assert 0 < int(bad.sum()) < p.t or window


@pytest.mark.gpu
@pytest.mark.parametrize("many,kind,hq,hkv,d", [(False, *x) for x in SHAPES] + [(True, *x) for x in MANY_SHAPES])
@pytest.mark.parametrize("past,new,window,sinks", [([900], [40], 0, 0), ([900], [40], 300, 40), ([20011], [3], 0, 0), ([0], [130], 0, 0)])
def test_infinities_of_v_do_not_depend_on_their_weights(gpu, many, kind, hq, hkv, d, past, new, window, sinks):
    """Scores of several hundred at one key leave the others weights of 0.  An
    infinity or NaN among those values still reaches each row that sees it, in
    masked and unmasked sub-tiles, in pieces of a split request and in either
    kernel; two infinities of different signs give NaN."""
    import torch
    kw = dict(window=window, sinks=sinks) if window else {}
    p = _Many(gpu, past, new, hq, hkv, d, kind, 16, seed=3, window=window) if many else _Paged(gpu, past, new, hq, hkv, d, kind, 16, seed=3)
    total, g = past[0] + new[0], hq // hkv
    big = total - new[0] - 5 if past[0] else 2  # the key that takes all weight of the rows that see it
    place = lambda j: (int(p.table[0, j // 16]), j % 16)  # noqa: E731
    p.q[: new[0]] = p.q[: new[0]].sign()
    p.k[p.table[0, : -(-total // 16)].long()] = 0.0
    p.k[place(big)] = (25 * p.q[0, ::g].float()).to(p.k.dtype)
    p.q[: new[0]] = p.q[:1, ::g].repeat_interleave(g, 1)  # every head of a group scores alike
    rows = torch.arange(past[0], total)
    sees = lambda j: (j <= rows) & ((window == 0) | (j > rows - window) | (j < sinks))  # noqa: E731
    values = {0: (math.inf, 3), min(100, total - 3): (-math.inf, 5), total - 20: (math.nan, 7), total - 2: (math.inf, 9), big - 1: (math.inf, 11), big + 1: (-math.inf, 11)}
    held = {}
    clean = p.run(**kw)
    p.check(clean, **kw)
    for j, (x, col) in values.items():
        held[j] = p.v[place(j)].clone()
        p.v[place(j)][hkv - 1, col] = x
    out = p.run(**kw)
    want = clean[: new[0]].float().cpu()
    odd = torch.zeros_like(want)
    for j, (x, col) in values.items():
        odd[:, -g:, col] += torch.where(sees(j)[:, None], x, 0.0)
    got = out[: new[0]].float().cpu()
    assert bool(((got == odd) | (got.isnan() & odd.isnan()))[odd != 0].all())
    # (f32 walks keys again on the f32 unit where a row is not finite: within the bound of _Paged.check)
    _, size, big_score = p.exact(0, **kw)
    slack = 2.0 ** -18 * (1 + big_score) * size if kind == "f32" else torch.zeros_like(size)
    assert bool(((got.double() - want.double()).abs() <= slack)[odd == 0].all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,hq,hkv,d", [("bf16", 8, 2, 128), ("bf16", 4, 2, 256), ("f32", 4, 2, 128)])
def test_sums_that_overflow_stay_infinite(gpu, kind, hq, hkv, d):
    """Finite values whose sum passes the type: no value that is not finite is there, and the infinity stays."""
    import torch
    p = _Paged(gpu, [200], [3], hq, hkv, d, kind, 16, seed=5)
    p.q.zero_()
    p.v[..., 4] = 3.0e38
    out = p.run()
    assert bool((out[..., 4] == math.inf).all())
    p.v[..., 4] = out[..., 4] = 0.0
    p.check(out)


@pytest.mark.gpu
@pytest.mark.parametrize("many", [False, True])
def test_a_cache_of_nan_ends_in_time(gpu, many):
    """Nothing but NaN in V: every row is NaN, by way of the slow path of every tile."""
    p = (_Many if many else _Paged)(gpu, [3000, 10], [70, 1], 8, 2, 128, "bf16", 16, seed=5)
    p.v.fill_(math.nan)
    att = p.attention()
    att.plan(p.cu, p.lengths)
    assert bool(att(p.q, p.k, p.v, p.table).isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("many,kind,hq,hkv,d", [(False, *x) for x in SHAPES] + [(True, *x) for x in MANY_SHAPES])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_near_the_largest_that_are_exact(gpu, many, kind, hq, hkv, d, sign):
    """Equal scores of 2^27.5 (d = 128) or 2^28 (256) in size: a maximum is then off by
    up to 2^3 in the exponent, the same for all keys of a row, and the rows are means."""
    import torch
    p = (_Many if many else _Paged)(gpu, [700], [90], hq, hkv, d, kind, 16, seed=6)
    p.q.fill_(2.0 ** 12)
    p.k.fill_(sign * 2.0 ** 12)
    out = p.run()[:90].double().cpu()
    v = p.keys(0, p.v).cpu().repeat_interleave(hq // hkv, 1)
    n = torch.arange(701, 791)[:, None, None]
    mean, size = v.cumsum(0)[700:] / n, v.abs().cumsum(0)[700:] / n
    # the weights of a row are equal, to half a step of bf16 where the two lane halves or pieces differ in their factor
    half = HALF[kind]
    assert bool(((out - mean).abs() <= (2 * half if kind == "bf16" else 2.0 ** -18) * size + half * mean.abs() * 1.01).all())


@pytest.mark.gpu
@pytest.mark.parametrize("many,kind,hq,hkv,d", [(False, "bf16", 8, 2, 128), (False, "bf16", 4, 2, 256), (False, "f32", 4, 2, 128), (True, "bf16", 8, 2, 128),
                                                (True, "bf16", 4, 2, 256)])
def test_infinities_of_v_in_caches_of_other_strides(gpu, many, kind, hq, hkv, d):
    """Head-major caches, out inside a larger buffer, in place of q, infinities of the first and the last KV head."""
    import torch
    for window, sinks in ((0, 0), (70, 5)):
        kw = dict(window=window, sinks=sinks) if window else {}
        extra = dict(window=window) if many else {}
        p = (_Many if many else _Paged)(gpu, [600, 20], [100, 1], hq, hkv, d, kind, 32, seed=7, head_major=True, **extra)
        clean = p.run(**kw)
        rows, g = torch.arange(600, 700, device=gpu), hq // hkv
        for j, head in ((3, 0), (590, hkv - 1), (640, 0), (698, hkv - 1)):
            page, off = int(p.table[0, j // 32]), j % 32
            held = p.v[page, off, head, d - 1].clone()
            p.v[page, off, head, d - 1] = -math.inf
            out = torch.full((p.t, 2 * hq, d), 5.0, dtype=p.q.dtype, device=gpu)[:, ::2]
            p.run(out=out, **kw)
            q = p.q.clone()
            assert torch.equal(p.run(out=p.q, **kw)[:100], out[:100])
            p.q = q
            p.v[page, off, head, d - 1] = held
            sees = (j <= rows) & ((window == 0) | (j > rows - window) | (j < sinks))
            assert bool((out[:100][sees][:, head * g: (head + 1) * g, d - 1] == -math.inf).all())
            got, want = out[:101].clone(), clean[:101].clone()
            got[:100][sees, head * g: (head + 1) * g, d - 1] = 0
            want[:100][sees, head * g: (head + 1) * g, d - 1] = 0
            assert bool(got.isfinite().all()) and (kind == "f32" or torch.equal(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("requests,room", [(20, 1500), (300, 6000)])
def test_tables_of_many_workgroups_in_a_graph(gpu, requests, room):
    """One captured step in place, replayed while requests grow, end and come back,
    with eager steps and other work between the replays."""
    import torch
    rng = random.Random(requests)
    s = _Tables(gpu, [rng.randint(0, 60) for _ in range(requests)], 16, 30, requests * 20, seed=3, max_tokens=room)
    new = s.t([0] * requests)

    def step():
        cev_hip.paged_tables(s.lengths, new, s.table, 16, s.cu, s.pos, s.slots, free=s.free, ring=s.ring)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(8):
        add = [rng.choice([-1, 0, 1, 20]) for _ in range(requests)]
        want = s.expect(add)
        new.copy_(s.t(add))
        if k % 3 == 2:
            step()
        else:
            graph.replay()
        torch.randn(1000, 1000, device=gpu).sum()
        torch.cuda.synchronize()
        s.check(want, k)
