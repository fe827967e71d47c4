"""GPU tests of the attention block (norm + rotation, paged cache store and load, attention of one token), through the
public Python entry points, against 64-bit restatements of the formulas.

Tolerances. u = 2^-8 is half a step of bf16 relative to the value, h = 2^-11 of fp16, e = 2^-24 of f32.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U, H, E = 2.0 ** -8, 2.0 ** -11, 2.0 ** -24
BF, F64 = torch.bfloat16, torch.float64


@pytest.fixture(scope="module", autouse=True)
def _need_gpu(vpq):
    assert torch.cuda.is_available(), "the -m gpu tests need a CUDA device"
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()
    assert vpq.ops.device_status() == 0


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def indexes_reported(vpq):
    """The kinds of index that were out of range since the last call."""
    import ctypes as C
    d = C.c_uint32(0)
    rc = vpq.lib().vpq_device_status(torch.cuda.current_stream().cuda_stream, C.byref(d))
    assert rc in (0, 8) and (rc == 0) == (d.value == 0)
    return d.value & 0xFF


# ------------------------------------------------------------------------------------- norm and rotation
def angles(rows, rot, g):
    a = torch.rand(rows, rot // 2, generator=g, device="cuda", dtype=F64) * 6.3
    return torch.cat([a.cos(), a.sin()], 1).float()


def ref_norm_rope(x, w, table, pos, eps, interleaved):
    """64-bit result, and the size of what each output value is the sum of."""
    y = x.to(F64)
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.to(F64)
    if table is None:
        return y, y.abs()
    rot = table.shape[1]
    row = table[pos].to(F64)[:, None]
    c, s = row[..., : rot // 2], row[..., rot // 2:]
    out, size = y.clone(), y.abs()
    if interleaved:
        ia, ib = torch.arange(0, rot, 2), torch.arange(1, rot, 2)
    else:
        ia, ib = torch.arange(0, rot // 2), torch.arange(rot // 2, rot)
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return out, size


def check_norm_rope(got, want, size):
    # one rounding to bf16, and before it in f32: the sum of squares (its terms are positive: D / 8 + 8 steps of e
    # at most, halved by the root), rsqrt (2 steps), two products, two products and a sum in the rotation
    tol = U * want.abs() * (1 + U) + 40 * E * size + 2.0 ** -133
    bad = (got.to(F64) - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got.to(F64) - want).abs() / tol).max()))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("M,hq,hkv", [(1, 32, 8), (3, 7, 1), (17, 5, 3), (300, 40, 40)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope(vpq, D, M, hq, hkv, interleaved):
    g = gen(D + M + hq)
    for rot in (D, 16, D // 2 if D > 32 else 16, 0, D - 16):
        q, k = (normal(g, M, hq, D) * 3).to(BF), (normal(g, M, hkv, D) * 0.01).to(BF)
        qw, kw = normal(g, D).to(BF), (1 + 0.1 * normal(g, D)).to(BF)
        table = angles(77, rot, g) if rot else None
        pos = torch.randint(0, 77, (M,), generator=g, device="cuda", dtype=torch.int32) if rot else None
        qo, ko = vpq.ops.qk_norm_rope(q, k, qw, kw, table, pos, eps=1e-5, interleaved=interleaved)
        p = pos.long() if rot else None
        check_norm_rope(qo, *ref_norm_rope(q, qw, table, p, 1e-5, interleaved))
        check_norm_rope(ko, *ref_norm_rope(k, kw, table, p, 1e-5, interleaved))


def test_norm_rope_without_norm_without_positions_and_in_place(vpq):
    g = gen(5)
    M, hq, hkv, D = 33, 6, 2, 128
    rows = normal(g, M, hq + 2 * hkv + 1, D).to(BF)  # q | k | v and a gap: strided views of one buffer
    q, k = rows[:, :hq], rows[:, hq:hq + hkv]
    table = angles(M + 4, 64, g)
    qw = normal(g, D).to(BF)
    at = torch.arange(M, device="cuda")
    want_q = ref_norm_rope(q.clone(), qw, table, at, 1e-6, True)
    want_k = ref_norm_rope(k.clone(), None, table, at, 1e-6, True)  # k without a norm
    rest = rows[:, hq + hkv:].clone()
    qo, ko = vpq.ops.qk_norm_rope(q, k, qw, None, table, None, interleaved=True, q_out=q, k_out=k)
    assert qo.data_ptr() == q.data_ptr() and ko.data_ptr() == k.data_ptr()
    check_norm_rope(q, *want_q)
    check_norm_rope(k, *want_k)
    assert torch.equal(rows[:, hq + hkv:], rest)
    # nothing to do at all: a copy
    z = normal(g, 2, 3, 64).to(BF)
    a, b = vpq.ops.qk_norm_rope(z, z)
    assert torch.equal(a, z) and torch.equal(b, z)
    # no rows
    a, b = vpq.ops.qk_norm_rope(z[:0], z[:0])
    assert a.shape == (0, 3, 64)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,hq,hkv", [(64, 32, 8), (64, 38, 3), (128, 32, 8), (128, 17, 5), (256, 14, 2)])
def test_norm_rope_of_a_prompt(vpq, D, hq, hkv, interleaved):
    """Rows of a prompt, out of place and in place: launches that take several heads at a time (2049 rows are enough for
    that at each of these head sizes) against the formula, and against the same rows a few at a time."""
    g = gen(D + hq)
    M = 2049
    assert M * (hq + hkv) > 148 * 8 * (256 // (D // 8)) * 2
    rows = normal(g, M, hq + 2 * hkv, D).to(BF)
    q, k = rows[:, :hq], rows[:, hq:hq + hkv]
    qw, kw = normal(g, D).to(BF), (1 + 0.1 * normal(g, D)).to(BF)
    for rot, by_position in ((D, True), (D // 2, True), (D, False)):
        table = angles(5000, rot, g)
        pos = torch.randint(0, 5000, (M,), generator=g, device="cuda", dtype=torch.int32) if by_position else None
        at = pos.long() if by_position else torch.arange(M, device="cuda")
        qo, ko = vpq.ops.qk_norm_rope(q, k, qw, kw, table, pos, interleaved=interleaved)
        check_norm_rope(qo, *ref_norm_rope(q, qw, table, at, 1e-6, interleaved))
        check_norm_rope(ko, *ref_norm_rope(k, kw, table, at, 1e-6, interleaved))
        for m in (0, 1000, M - 5):
            few = slice(m, m + 5)
            a, b = vpq.ops.qk_norm_rope(q[few], k[few], qw, kw, table if by_position else table[few].contiguous(),
                                        pos[few].contiguous() if by_position else None, interleaved=interleaved)
            assert torch.equal(a, qo[few]) and torch.equal(b, ko[few])
        here = rows.clone()
        vpq.ops.qk_norm_rope(here[:, :hq], here[:, hq:hq + hkv], qw, kw, table, pos, interleaved=interleaved,
                             q_out=here[:, :hq], k_out=here[:, hq:hq + hkv])
        assert torch.equal(here[:, :hq], qo) and torch.equal(here[:, hq:hq + hkv], ko)
        assert torch.equal(here[:, hq + hkv:], rows[:, hq + hkv:])


def test_rows_with_a_position_outside_are_left_as_they_were(vpq):
    g = gen(6)
    M, D = 9, 64
    q, k = normal(g, M, 4, D).to(BF), normal(g, M, 2, D).to(BF)
    table = angles(10, D, g)
    pos = torch.tensor([0, -1, 9, 3, -7, 1, 2, -2147483648, 5], dtype=torch.int32, device="cuda")
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    vpq.ops.qk_norm_rope(q, k, None, None, table, pos, q_out=qo, k_out=ko)
    dead = pos < 0
    assert (qo[dead] == 7).all() and (ko[dead] == 7).all()
    live = ~dead
    check_norm_rope(qo[live], *ref_norm_rope(q[live], None, table, pos[live].long(), 1e-6, False))
    assert indexes_reported(vpq) == 0
    pos[0], pos[3] = 10, 2147483647
    qo.fill_(7.0)
    vpq.ops.qk_norm_rope(q, k, None, None, table, pos, q_out=qo, k_out=ko)
    assert (qo[0] == 7).all() and (qo[3] == 7).all()
    assert indexes_reported(vpq) == 4
    assert indexes_reported(vpq) == 0


# ------------------------------------------------------------------------------------- the cache
def layouts(vpq, kind, pages, ps, heads, D, bits):
    """Caches of the same shape over different memory."""
    dt = BF if bits == 16 else torch.uint8
    pair = (D // 64, 2)
    fill = float("nan") if bits == 16 else 0xEE
    mk = lambda *s: torch.full(s, fill, dtype=dt, device="cuda")  # noqa: E731
    sc = lambda *s: torch.full(s, float("nan"), dtype=BF, device="cuda")  # noqa: E731
    if kind == "dense":
        t = [mk(pages, heads, ps, D), mk(pages, heads, ps, D)]
        s = [sc(pages, heads, ps, *pair), sc(pages, heads, ps, *pair)]
    elif kind == "token_major":
        t = [mk(pages, ps, heads, D).transpose(1, 2) for _ in range(2)]
        s = [sc(pages, ps, heads, *pair).transpose(1, 2) for _ in range(2)]
    else:  # keys and values of a page side by side, rows of a wider buffer
        pool = mk(pages, 2, heads, ps, D + 64)
        t = [pool[:, i, :, :, :D] for i in range(2)]
        spool = sc(pages, 2, heads, ps, *pair)
        s = [spool[:, i] for i in range(2)]
    return vpq.ops.PagedKVCache(*t, *(s if bits == 8 else []))


def held(cache):
    """64-bit values of the whole cache [pages, heads, page, D] (k, v)."""
    got = []
    for x, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        y = x.to(F64)
        if s is not None:
            p = s.to(F64).repeat_interleave(64, dim=3)
            y = y * p[..., 0] + p[..., 1]
        got.append(y)
    return got


def at_slots(x, slots, ps):
    return x[slots // ps, :, slots % ps]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kind", ["dense", "token_major", "pool"])
@pytest.mark.parametrize("bits", [16, 8])
def test_store_and_load(vpq, D, kind, bits):
    g = gen(D + bits)
    for M, heads, ps in ((1, 8, 16), (37, 3, 48), (400, 2, 32)):
        pages = -(-M // ps) + 3
        c = layouts(vpq, kind, pages, ps, heads, D, bits)
        rows = torch.randperm(pages * ps, generator=g, device="cuda")[:M]
        k = (normal(g, M, heads, D) * (1 + 20 * (torch.rand(D, generator=g, device="cuda") < 0.05)) + 3).to(BF)
        v = (normal(g, M, heads, D) * 1e-3).to(BF)
        if M > 30:
            k[3] = 1.5                     # groups of equal values
            v[4] = 0.0
            v[5] = torch.where(torch.arange(D, device="cuda") % 2 == 0, 0.0, -0.0).to(BF)
            k[6] = (20.0 + 0.25 * torch.rand(heads, D, generator=g, device="cuda")).to(BF)   # offset >> spread
            v[7] = (normal(g, heads, D) * 1e-38).to(BF)
            k[8] = (normal(g, heads, D) * 1e37).to(BF)
        before = [t.clone() for t in (c.k, c.v)]
        slots = rows.clone()
        if M > 1:
            slots[-1] = -1
        vpq.ops.kv_store(k, v, c, slots)
        kl, vl = vpq.ops.kv_load(c, slots)
        live = slots >= 0
        for x, y, whole in ((k, kl, held(c)[0]), (v, vl, held(c)[1])):
            z = at_slots(whole, slots[live], ps)
            if bits == 16:
                assert torch.equal(y[live], x[live])
            else:
                pairs = at_slots(c.k_scales if x is k else c.v_scales, slots[live], ps).to(F64)
                s = pairs[..., 0].repeat_interleave(64, dim=2)
                # rint of a quotient made with three f32 roundings of a number up to 255: within half a step and
                # 255 * 3 e of the value; the scale's own rounding up may miss by one f32 step
                assert ((z - x[live].to(F64)).abs() <= s * (0.5 + 255 * 4 * E)).all()
                # load: one f32 rounding of s c + b, one to bf16
                assert ((y[live].to(F64) - z).abs() <= U * z.abs() * (1 + U) + 2 * E * (s * 255 + pairs[..., 1].abs().repeat_interleave(64, dim=2))).all()
                # and the pair is what the definition says: bias the minimum itself (it is a bf16 number)
                grp = x[live].to(F64).reshape(x[live].shape[0], heads, D // 64, 64)
                assert torch.equal(pairs[..., 1], grp.amin(-1))
                step = (grp.amax(-1) - grp.amin(-1)) / 255
                assert (pairs[..., 0] >= step * (1 - 4 * E)).all()
                assert (pairs[..., 0] <= torch.maximum(step * (1 + 2 * U + 4 * E), torch.full_like(step, 2.0 ** -126))).all()
            assert (y[~live] == 0).all()
        # what no slot names is untouched
        hit = torch.zeros(pages * ps, dtype=torch.bool, device="cuda")
        hit[slots[live]] = True
        hit = hit.view(pages, 1, ps, 1)
        for t, b in zip((c.k, c.v), before):
            same = (t == b) | (t.isnan() & b.isnan()) if bits == 16 else t == b
            assert (same | hit).all()
    assert indexes_reported(vpq) == 0


def test_a_group_with_a_nan_or_infinity_reads_back_as_nan(vpq):
    c = layouts(vpq, "dense", 2, 16, 2, 128, 8)
    k = torch.ones(3, 2, 128, dtype=BF, device="cuda")
    v = k.clone()
    k[0, 0, 5], k[1, 1, 70], v[2, 0, 127] = float("nan"), float("inf"), -float("inf")
    v[1, 0, 0], v[1, 0, 1] = 3.3e38, -3.3e38
    slots = torch.tensor([1, 17, 30], device="cuda")
    vpq.ops.kv_store(k, v, c, slots)
    kl, vl = vpq.ops.kv_load(c, slots)
    bad_k = torch.zeros(3, 2, 2, dtype=torch.bool, device="cuda")
    bad_k[0, 0, 0] = bad_k[1, 1, 1] = True
    bad_v = torch.zeros_like(bad_k)
    bad_v[2, 0, 1] = bad_v[1, 0, 0] = True
    assert torch.equal(kl.isnan(), bad_k.repeat_interleave(64, 2))
    assert torch.equal(vl.isnan(), bad_v.repeat_interleave(64, 2))
    assert (kl[~kl.isnan()] == 1).all() and (vl[~vl.isnan()] == 1).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_slots_outside_are_skipped_and_reported(vpq, bits):
    c = layouts(vpq, "dense", 3, 16, 2, 64, bits)
    before = [t.clone() for t in (c.k, c.v)]
    k = torch.ones(3, 2, 64, dtype=BF, device="cuda")
    slots = torch.tensor([48, 1 << 40, -(1 << 40)], device="cuda")
    vpq.ops.kv_store(k, k, c, slots)
    assert indexes_reported(vpq) == 2
    for t, b in zip((c.k, c.v), before):
        assert ((t == b) | ((t != t) & (b != b))).all()
    kl, vl = vpq.ops.kv_load(c, slots)
    assert (kl == 0).all() and (vl == 0).all()
    assert indexes_reported(vpq) == 2


def test_reports_of_two_streams_are_both_seen(vpq):
    """A report that arrives while another is read back and cleared is in that call's answer or in the next one's,
    whenever it arrives (here: over a hundred microseconds, half a microsecond apart)."""
    side = torch.cuda.Stream()
    c = layouts(vpq, "dense", 3, 16, 2, 64, 16)
    k = torch.ones(1, 2, 64, dtype=BF, device="cuda")
    table = torch.ones(4, 64, device="cuda")
    slot, pos = torch.tensor([48], device="cuda"), torch.tensor([4], dtype=torch.int32, device="cuda")
    out = torch.empty_like(k)
    for i in range(600):
        vpq.ops.kv_store(k, k, c, slot)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(1000 * (i % 200))
        vpq.ops.qk_norm_rope(k, k, None, None, table, pos, q_out=out, k_out=out.clone(), stream=side)
        first = indexes_reported(vpq)
        side.synchronize()
        second = indexes_reported(vpq)
        assert first & 2 and first | second == 2 | 4, (i, first, second)
        assert indexes_reported(vpq) == 0


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("M,hq,hkv,D,rot,interleaved", [(1, 32, 8, 128, 128, False), (5, 7, 1, 64, 32, True),
                                                        (130, 6, 3, 256, 64, False), (700, 32, 8, 128, 128, False)])
def test_store_pass_is_norm_rope_then_store(vpq, bits, M, hq, hkv, D, rot, interleaved):
    g = gen(M + D)
    rows = normal(g, M, hq + 2 * hkv, D).to(BF)
    q, k, v = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:]
    qw, kw = normal(g, D).to(BF), normal(g, D).to(BF)
    table = angles(50, rot, g)
    pos = torch.randint(0, 50, (M,), generator=g, device="cuda", dtype=torch.int32)
    ps, pages = 32, -(-M // 32) + 1
    slots = torch.randperm(pages * ps, generator=g, device="cuda")[:M]
    if M > 4:
        slots[2] = -1      # q is made, nothing is stored
        pos[4] = -1        # the row is skipped altogether
    c = layouts(vpq, "token_major", pages, ps, hkv, D, bits)
    plain = layouts(vpq, "token_major", pages, ps, hkv, D, bits)
    qo = vpq.ops.qkv_norm_rope_store(q, k, v, qw, kw, table, pos, c, slots, interleaved=interleaved,
                                     q_out=torch.full_like(q, 9.0))
    q2, k2 = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
    vpq.ops.qk_norm_rope(q, k, qw, kw, table, pos, interleaved=interleaved, q_out=q2, k_out=k2)
    assert torch.equal(qo, q2)
    use = slots.clone()
    if M > 4:
        use[4] = -1
    vpq.ops.kv_store(k2, v, plain, use)
    same = lambda a, b: bool(((a == b) | ((a != a) & (b != b))).all())  # noqa: E731
    assert same(c.v, plain.v)
    if bits == 16:
        assert same(c.k, plain.k)
    else:
        assert same(c.v_scales, plain.v_scales)
        live = use >= 0
        want, size = ref_norm_rope(k[live], kw, table, pos[live].long(), 1e-6, interleaved)
        z = at_slots(held(c)[0], use[live], ps)
        s = at_slots(c.k_scales, use[live], ps).to(F64)[..., 0].repeat_interleave(64, dim=2)
        # codes of the unrounded f32 keys: half a step, and the keys' own f32 error
        assert ((z - want).abs() <= s * (0.5 + 255 * 4 * E) + 40 * E * size).all()
        untouched = torch.ones(pages * ps, dtype=torch.bool, device="cuda")
        untouched[use[live]] = False
        assert same(at_slots(c.k, untouched.nonzero().squeeze(1), ps), at_slots(plain.k, untouched.nonzero().squeeze(1), ps))


# ------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bits", [16, 8])
def test_many_rows_as_few(vpq, D, bits):
    """Launches that take several heads at a time give what small ones give, for head counts that do and do not divide."""
    g = gen(31)
    for heads, kind in ((8, "dense"), (8, "token_major"), (4, "shared"), (11, "dense")):
        M, ps = 7003, 48
        c = layouts(vpq, kind, 160, ps, heads, D, bits)
        k, v = (normal(g, M, heads, D).to(BF) for _ in range(2))
        slots = torch.randperm(160 * ps, generator=g, device="cuda")[:M].contiguous()
        slots[5], slots[M - 1], slots[4000] = -1, -7, 160 * ps + 3
        vpq.ops.kv_store(k, v, c, slots)
        kl, vl = vpq.ops.kv_load(c, slots)
        for m in range(0, M, 500):
            few = slice(m, min(m + 500, M))
            d = layouts(vpq, kind, 160, ps, heads, D, bits)
            vpq.ops.kv_store(k[few], v[few], d, slots[few].contiguous())
            a, b = vpq.ops.kv_load(d, slots[few].contiguous())
            assert torch.equal(a, kl[few]) and torch.equal(b, vl[few])
            a, b = vpq.ops.kv_load(c, slots[few].contiguous())
            assert torch.equal(a, kl[few]) and torch.equal(b, vl[few])
        for bad in (5, M - 1, 4000):
            assert (kl[bad] == 0).all() and (vl[bad] == 0).all()
        assert indexes_reported(vpq) == 2


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("hq,hkv,D,rot,interleaved", [(32, 8, 128, 128, False), (14, 2, 64, 32, True),
                                                      (16, 2, 256, 64, False), (11, 11, 128, 128, True)])
def test_many_rows_of_the_pass_as_few(vpq, bits, hq, hkv, D, rot, interleaved):
    """The same of the pass into the cache: how rows are dealt changes nothing."""
    g = gen(32)
    M, ps = 6003, 16
    rows = normal(g, M, hq + 2 * hkv, D).to(BF)
    q, k, v = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:]
    qw, kw = normal(g, D).to(BF), (1 + 0.1 * normal(g, D)).to(BF)
    table = angles(512, rot, g)
    pos = torch.randint(0, 512, (M,), generator=g, device="cuda", dtype=torch.int32)
    slots = torch.randperm(400 * ps, generator=g, device="cuda")[:M].contiguous()
    pos[17], slots[3000], slots[M - 1] = -1, -1, -5
    live = (pos >= 0) & (slots >= 0)

    def run(take, c):
        n = len(range(*take.indices(M)))
        out = torch.full((n, hq, D), 7.0, dtype=BF, device="cuda")
        vpq.ops.qkv_norm_rope_store(q[take], k[take], v[take], qw, kw, table, pos[take].contiguous(), c,
                                    slots[take].contiguous(), interleaved=interleaved, q_out=out)
        return out

    c, d = (layouts(vpq, "dense", 400, ps, hkv, D, bits) for _ in range(2))
    whole = run(slice(0, M), c)
    for m in range(0, M, 300):
        assert torch.equal(run(slice(m, min(m + 300, M)), d), whole[m:m + 300])
    assert (whole[17] == 7).all()
    for a, b in zip(vpq.ops.kv_load(c, slots), vpq.ops.kv_load(d, slots)):
        assert torch.equal(a[live], b[live])
    check_norm_rope(whole[pos >= 0], *ref_norm_rope(q[pos >= 0], qw, table, pos[pos >= 0].long(), 1e-6, interleaved))
    for x, y in ((c.k, d.k), (c.v, d.v)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert indexes_reported(vpq) == 0


def filled(vpq, g, kind, lens, ps, heads, D, bits, gain=1.0, spare=2):
    """A cache with random tokens, NaN everywhere else, and the page table: columns past a sequence's pages hold
    numbers that must never be followed."""
    need = [max(0, -(-n // ps)) for n in lens]
    pages = sum(need) + spare
    c = layouts(vpq, kind, pages, ps, heads, D, bits)
    place = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(lens), max(max(need), 1) + 1), 1 << 30, dtype=torch.int32, device="cuda")
    table[:, -1] = -5
    used = 0
    for b, n in enumerate(need):
        table[b, :n] = place[used:used + n]
        used += n
        if lens[b] <= 0:
            continue
        t = torch.arange(lens[b], device="cuda")
        slots = table[b, t // ps].long() * ps + t % ps
        off = 2 * normal(g, heads, D)
        vpq.ops.kv_store((gain * (normal(g, lens[b], heads, D) + off)).to(BF), (normal(g, lens[b], heads, D) + off).to(BF),
                         c, slots)
    return c, table


def ref_attention(q, c, table, lens, scale, window):
    """64-bit output and its tolerance."""
    ps, D = c.page_size, c.head_dim
    k_all, v_all = held(c)
    B, hq, _ = q.shape
    per = hq // c.kv_heads
    out, tol = torch.zeros(B, hq, D, dtype=F64, device="cuda"), torch.zeros(B, hq, D, dtype=F64, device="cuda")
    for b, n in enumerate(lens):
        first = max(0, n - window) if window else 0
        if n <= first:
            continue
        t = torch.arange(first, n, device="cuda")
        page = table[b, t // ps].long()
        k, v = k_all[page, :, t % ps], v_all[page, :, t % ps]
        for h in range(c.kv_heads):
            x = q[b, h * per:(h + 1) * per].to(F64)
            s = x @ k[:, h].T * scale
            p = torch.softmax(s, -1)
            o = p @ v[:, h]
            size = p @ v[:, h].abs()
            # a score: D products added in f32 (the product unit may cut instead of round: two steps each), for 8 bits also of
            # centred codes and of the biases, whose terms are no larger than three times the values'; then the
            # scale, the maximum's subtraction and 2^x (2 steps of the result)
            mag = 3 if c.bits == 8 else 1
            eps = float((scale * mag * (x.abs() @ k[:, h].abs().T)).max()) * (2 * D + 16) * E + float(s.abs().max()) * 8 * E + 8 * E
            # the weights' rounding: to bf16, or p s to fp16 over centred codes (|c - 128| s and the bias term are
            # each within three times the largest value of the group)
            if c.bits == 16:
                w = 2 * U * size
            else:
                big = v[:, h].abs().reshape(len(t), D // 64, 64).amax(-1).repeat_interleave(64, -1)
                w = 3 * (H + 64 * E) * (p @ big) + 2.0 ** -39 * 128 * big.max()
            out[b, h * per:(h + 1) * per] = o
            tol[b, h * per:(h + 1) * per] = U * o.abs() * (1 + U) + 1.01 * (w + 2 * eps * size) + 16 * E * size
    return out, tol


def check_attention(vpq, q, c, table, lens, scale=None, window=0, **kw):
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = vpq.ops.paged_attention(q, c, table, dl, scale=scale, window=window, **kw)
    want, tol = ref_attention(q, c, table, lens, scale or 1 / math.sqrt(c.head_dim), window)
    err = (got.to(F64) - want).abs()
    assert (err <= tol).all(), (float((err / tol.clamp(min=1e-300)).max()), int((err > tol).sum()), got.isnan().sum())
    again = vpq.ops.paged_attention(q, c, table, dl, scale=scale, window=window, **kw)
    assert torch.equal(got, again)
    return got


@pytest.mark.parametrize("D", [128, 64, 256])
@pytest.mark.parametrize("bits", [16, 8])
def test_attention_lengths(vpq, D, bits):
    """One sequence: every length around a unit and a page; then a batch of them, empty ones among them."""
    g = gen(D + bits)
    for n in (1, 2, 15, 16, 17, 31, 33, 47, 49, 128, 129, 255, 1000):
        c, table = filled(vpq, g, "dense", [n], 48, 2, D, bits)
        check_attention(vpq, normal(g, 1, 8, D).to(BF), c, table, [n])
    lens = [0, 1, 0, 0, 700, 16, 33, 0, 5, 48, 2000, 0]
    c, table = filled(vpq, g, "dense", lens, 16, 2, D, bits)
    out = check_attention(vpq, normal(g, len(lens), 8, D).to(BF), c, table, lens)
    assert (out[[0, 2, 3, 7, 11]] == 0).all()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D,hq,hkv", [(128, 32, 8), (128, 1, 1), (128, 5, 1), (128, 7, 1), (128, 18, 2), (128, 16, 1),
                                      (128, 17, 1), (128, 71, 1), (64, 12, 12), (64, 9, 1), (64, 40, 1), (256, 8, 1),
                                      (256, 9, 1), (256, 16, 1), (256, 6, 3)])
def test_attention_head_layouts(vpq, bits, D, hq, hkv):
    g = gen(hq * 100 + hkv)
    lens = [97, 3, 0, 260, 16]
    c, table = filled(vpq, g, "token_major", lens, 32, hkv, D, bits)
    check_attention(vpq, normal(g, len(lens), hq, D).to(BF), c, table, lens)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("window", [1, 5, 16, 17, 100, 5000])
def test_attention_window(vpq, bits, window):
    g = gen(window)
    lens = [1, 4, 17, 16, 120, 700, 0]
    c, table = filled(vpq, g, "pool", lens, 16, 2, 128, bits)
    # pages that lie wholly before the window may be gone
    for b, n in enumerate(lens):
        gone = max(0, n - window) // 16
        table[b, :gone] = -9
    want_table = table.clone()
    want_table[want_table < 0] = 0
    q = normal(g, len(lens), 8, 128).to(BF)
    got = vpq.ops.paged_attention(q, c, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), window=window)
    want, tol = ref_attention(q, c, want_table, lens, 1 / math.sqrt(128), window)
    assert ((got.to(F64) - want).abs() <= tol).all()
    assert indexes_reported(vpq) == 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("window", [1, 17, 1000])
def test_attention_window_that_cuts_many_sequences(vpq, bits, D, window):
    """Windows that begin inside of sequences, with more (sequence, key head) pairs than SMs: one line of units from window
    to window, whose runs begin and end anywhere in them."""
    g = gen(window + D)
    lens = [0, 1, 2, 16, 17, 999, 1000, 1001, 1016, 1017, 2500, 3000]
    lens += torch.randint(0, 2000, (28,), generator=g, device="cuda").tolist()
    hkv, ps = 4, 48
    assert len(lens) * hkv > 148
    c, table = filled(vpq, g, "dense", lens, ps, hkv, D, bits)
    want_table = table.clone()
    for b, n in enumerate(lens):  # pages that lie wholly before the window may be gone
        table[b, :max(0, n - window) // ps] = -9
    q = normal(g, len(lens), 2 * hkv, D).to(BF)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = vpq.ops.paged_attention(q, c, table, dl, window=window)
    want, tol = ref_attention(q, c, want_table, lens, 1 / math.sqrt(D), window)
    err = (got.to(F64) - want).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-300)).max())
    assert indexes_reported(vpq) == 0


def count_tokens(vpq, g, bits, D, hkv, per, lens, window, first=0):
    """Attention that counts: queries of 0 give every token the weight 1, and key head h has a 1 only in tokens 16 i + r,
    r = (first + h) % 16, there in column i % D. Every output is a small number of tokens over the window's length, so one
    token that is lost or taken twice shows."""
    ps, B = 48, len(lens)
    need = [-(-n // ps) for n in lens]
    pages = sum(need)
    c = layouts(vpq, "dense", pages, ps, hkv, D, bits)
    place = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((B, max(need)), 1 << 30, dtype=torch.int32, device="cuda")
    want = torch.zeros(B, hkv, D, dtype=F64, device="cuda")
    used = 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = place[used:used + need[b]]
        used += need[b]
        t = torch.arange(n, device="cuda")
        r = (first + torch.arange(hkv, device="cuda")) % 16
        v = torch.zeros(n, hkv, D, dtype=BF, device="cuda")
        v[t[:, None], torch.arange(hkv, device="cuda")[None], (t // 16 % D)[:, None]] = (t[:, None] % 16 == r[None]).to(BF)
        vpq.ops.kv_store(normal(g, n, hkv, D).to(BF), v, c, table[b, t // ps].long() * ps + t % ps)
        lo = max(0, n - window) if window else 0
        # what a 1 reads back as: 254 times 1 / 255 rounded up to bf16, if the cache has 8 bits
        one = 254 * 0.00393676757812 if bits == 8 else 1.0
        want[b] = v[lo:].to(F64).sum(0) * one / (n - lo)
    got = vpq.ops.paged_attention(torch.zeros(B, hkv * per, D, dtype=BF, device="cuda"), c, table,
                                  torch.tensor(lens, dtype=torch.int32, device="cuda"), window=window)
    # One rounding to bf16; in f32 the sum of weights is exact and its reciprocal and a product are two roundings. 8 bits: the
    # two sums of 128 s (at most 0.51) over a sixteenth of the tokens differ by the roundings of at most 200 additions of
    # two steps each, 200 * 2 E * 0.51 / 16 of the average.
    want = want.repeat_interleave(per, 1)
    tol = (U + 64 * E) * want + (16 * E if bits == 8 else 0)
    # a token more or less is more than that
    n = torch.tensor([min(n, window) if window else n for n in lens], device="cuda")
    assert (tol.amax((1, 2)) < 0.99 / n).all()
    err = (got.to(F64) - want).abs()
    assert (err <= tol).all(), (int((err > tol).sum()), float((err * n[:, None, None]).max()))


@pytest.mark.parametrize("per", [1, 5, 12])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bits", [16, 8])
def test_attention_counts_every_token_once(vpq, bits, D, per):
    """One key head over all CTAs, joined across all of them, for each place in sixteen; all sixteen at once; two sequences; a
    window that begins inside of a unit and a page."""
    g = gen(24 + D)
    for r in range(16):
        count_tokens(vpq, g, bits, D, 1, per, [40000 - 7 * r], 0, first=r)
    count_tokens(vpq, g, bits, D, 16, per, [40003], 0)
    count_tokens(vpq, g, bits, D, 16, per, [20011, 33333], 0)
    for window in (9001, 19990):
        count_tokens(vpq, g, bits, D, 1, per, [40000], window, first=window % 16)
        count_tokens(vpq, g, bits, D, 16, per, [20011, 33333], window)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bits", [16, 8])
def test_attention_counts_every_token_of_short_sequences_once(vpq, bits, D):
    """The same where a CTA has a whole sequence and key head, and where it has parts of several."""
    g = gen(25 + D)
    for n in (1, 15, 31, 32, 33, 47, 100, 333, 512):
        count_tokens(vpq, g, bits, D, 16, 4, [n, 1, n], 0)
    count_tokens(vpq, g, bits, D, 16, 4, [700 + 13 * i for i in range(20)], 0)
    count_tokens(vpq, g, bits, D, 16, 4, [700 + 13 * i for i in range(20)], 333)


def with_wide_tables(monkeypatch):
    """From here on page tables have room for thousands of tokens more than any sequence: how a call is split goes by
    that room, and the narrow tables of the tests above only ever give each sequence a CTA of its own."""
    narrow = filled

    def wide(*args, **kw):
        c, table = narrow(*args, **kw)
        return c, torch.nn.functional.pad(table, (0, 600), value=1 << 30)
    monkeypatch.setitem(globals(), "filled", wide)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D,hq,hkv", [(128, 32, 8), (128, 1, 1), (128, 5, 1), (128, 7, 1), (128, 18, 2), (128, 16, 1),
                                      (128, 17, 1), (128, 71, 1), (64, 12, 12), (64, 4, 1), (64, 9, 1), (64, 40, 1),
                                      (256, 8, 1), (256, 9, 1), (256, 16, 1), (256, 6, 3)])
def test_attention_head_layouts_wide_table(vpq, monkeypatch, bits, D, hq, hkv):
    with_wide_tables(monkeypatch)
    test_attention_head_layouts(vpq, bits, D, hq, hkv)


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_wide_tables(vpq, monkeypatch, bits):
    with_wide_tables(monkeypatch)
    for D in (64, 128, 256):
        test_attention_lengths(vpq, D, bits)
    test_attention_sharp_and_flat_scores(vpq, bits)
    test_attention_bad_pages_and_lengths(vpq, bits)
    test_attention_in_a_graph_follows_the_lengths(vpq, bits)
    if bits == 16:
        test_attention_nan_and_infinity_stay_with_their_sequence(vpq)
        test_attention_strided_queries_and_outputs(vpq)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("B,hkv", [(1, 1), (3, 8), (18, 8), (19, 8), (148, 1), (149, 1)])
def test_attention_full_tables(vpq, bits, B, hkv):
    """Sequences as long as their tables, empty and nearly empty ones beside them, at the sizes where the split changes."""
    g = gen(B)
    for n in (16, 496, 512, 528, 1024):
        lens = [n, 0, 1, n - 1, n // 2][:B] + [3] * (B - 5)
        c, table = filled(vpq, g, "dense", lens, 16, hkv, 128, bits)
        table = table[:, :n // 16].contiguous()
        check_attention(vpq, normal(g, B, 4 * hkv, 128).to(BF), c, table, lens)


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_long_and_uneven(vpq, bits):
    g = gen(77)
    lens = [30011, 1, 17, 4096, 0, 777]
    c, table = filled(vpq, g, "dense", lens, 64, 2, 128, bits)
    check_attention(vpq, normal(g, len(lens), 8, 128).to(BF), c, table, lens)
    # one key head alone, so that every CTA has a piece of the same head
    c, table = filled(vpq, g, "dense", [40000], 128, 1, 128, bits)
    check_attention(vpq, normal(g, 1, 4, 128).to(BF), c, table, [40000])


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_many_short_sequences(vpq, bits):
    """More sequences than threads look them up, most of them empty or of a token or two; a token of 1000 sequences at
    the same place of the same page is fine (a shared prefix)."""
    g = gen(3)
    B, D = 1000, 64
    c, table = filled(vpq, g, "dense", [160], 16, 1, D, bits)
    lens = torch.randint(0, 161, (B,), generator=g, device="cuda", dtype=torch.int32)
    lens[torch.rand(B, generator=g, device="cuda") < 0.5] = 0
    lens[0] = lens[-1] = 0
    check_attention(vpq, normal(g, B, 3, D).to(BF), c, table.expand(B, -1).contiguous(), lens.tolist())


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_sharp_and_flat_scores(vpq, bits):
    """Scores far apart (one token takes all), equal scores, and scores that keep growing along the sequence."""
    g = gen(9)
    c, table = filled(vpq, g, "dense", [500, 300], 16, 1, 128, bits, gain=20.0)
    check_attention(vpq, normal(g, 2, 4, 128).to(BF), c, table, [500, 300])
    check_attention(vpq, torch.zeros(2, 4, 128, dtype=BF, device="cuda"), c, table, [500, 300])
    check_attention(vpq, (normal(g, 2, 4, 128) * 1e-3).to(BF), c, table, [500, 300], scale=0.7)
    c, table = filled(vpq, g, "dense", [1], 16, 1, 128, bits)
    n = 400
    c2 = layouts(vpq, "dense", 26, 16, 1, 128, bits)
    t = torch.arange(n, device="cuda")
    k = torch.ones(n, 1, 128, device="cuda") * (t[:, None, None] / 16.0)
    vpq.ops.kv_store(k.to(BF), (normal(g, n, 1, 128) * (1.0 + t[:, None, None])).to(BF), c2, t)
    table2 = torch.arange(26, dtype=torch.int32, device="cuda")[None]
    check_attention(vpq, torch.ones(1, 8, 128, dtype=BF, device="cuda"), c2, table2, [n])


@pytest.mark.parametrize("gain", [1e-30, 1e-3, 1e4, 1e30])
def test_attention_8_bit_scales_of_any_size(vpq, gain):
    """Scales of keys and values over the whole range of bf16, and tokens whose value scales differ by far."""
    g = gen(11)
    n, D = 333, 128
    c = layouts(vpq, "dense", 21, 16, 2, D, 8)
    t = torch.arange(n, device="cuda")
    k = normal(g, n, 2, D) * gain
    v = normal(g, n, 2, D) * gain * 10.0 ** torch.randint(-3, 4, (n, 1, 1), generator=g, device="cuda").float()
    vpq.ops.kv_store(k.to(BF), v.to(BF), c, t)
    table = torch.arange(21, dtype=torch.int32, device="cuda")[None]
    q = (normal(g, 1, 8, D) / gain).to(BF)
    check_attention(vpq, q, c, table, [n], scale=0.1)


@pytest.mark.parametrize("D,per", [(64, 4), (128, 4), (128, 12), (256, 6)])
def test_attention_scales_of_either_sign(vpq, D, per):
    """Pages that another quantizer has filled: scales of either sign, zeros among them, any codes."""
    g = gen(26)
    lens = [200, 33, 1000]
    c, table = filled(vpq, g, "dense", lens, 16, 2, D, 8)
    for pairs in (c.k_scales, c.v_scales):
        s = normal(g, *pairs.shape[:-1]) * 0.01
        pairs[..., 0] = torch.where(torch.rand(s.shape, generator=g, device="cuda") < 0.1, torch.zeros_like(s), s).to(BF)
        pairs[..., 1] = normal(g, *pairs.shape[:-1]).to(BF)
    for pages in (c.k, c.v):
        pages.copy_(torch.randint(0, 256, pages.shape, generator=g, device="cuda", dtype=torch.uint8))
    check_attention(vpq, normal(g, 3, 2 * per, D).to(BF), c, table, lens)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("power", [120, 103, 60, -60, -112, -120])
def test_attention_large_scales_of_small_queries(vpq, bits, power):
    """Scores of ordinary size from a scale and queries that are not: only their product may bound the call."""
    g = gen(16)
    lens, D = [333, 40], 128
    c, table = filled(vpq, g, "dense", lens, 16, 2, D, bits)
    q = (normal(g, 2, 8, D) * 2.0 ** -power).to(BF)
    assert (q.abs() > 2.0 ** -126).float().mean() > 0.9
    check_attention(vpq, q, c, table, lens, scale=0.1 * 2.0 ** power)


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_averages_many_values(vpq, bits):
    """Equal weights over 131072 tokens, each warp adding up tens of thousands of them: what is left of the values is
    a three-hundredth of each, and must not drown in the sums it is taken from. (All sequences share the pages.)"""
    g = gen(12)
    n, D, B = 131072, 128, 600
    c = layouts(vpq, "dense", n // 64, 64, 1, D, bits)
    t = torch.arange(n, device="cuda")
    v = normal(g, n, 1, D).to(BF)
    vpq.ops.kv_store(v, v, c, t)
    q = torch.zeros(B, 1, D, dtype=BF, device="cuda")
    table = torch.arange(n // 64, dtype=torch.int32, device="cuda").expand(B, -1).contiguous()
    got = vpq.ops.paged_attention(q, c, table, torch.full((B,), n, dtype=torch.int32, device="cuda")).to(F64)[:, 0]
    want = held(c)[1].reshape(n, D).mean(0)
    # A weight is 1, exact in bf16. For 8 bits 2^15 s / 2^k is rounded to fp16: at most H, independently of the codes
    # (128 s is at most 5.5 / 255 * 128 here), so eight standard deviations of the mean; and each unit's products and
    # its sum are off by a few f32 steps of 255 s times its weights. bf16: a sum in f32, cut at each of 8192 steps.
    half = 128 * 11.0 / 255
    tol = U * want.abs() * (1 + U) + (8 * H * half / math.sqrt(n) + 16 * E * half if bits == 8 else 8192 * 2 * E * want.abs() + 16 * E * 5.5)
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


def test_attention_nan_and_infinity_stay_with_their_sequence(vpq):
    g = gen(13)
    lens = [40, 50, 60]
    c, table = filled(vpq, g, "dense", lens, 16, 1, 128, 16)
    q = normal(g, 3, 4, 128).to(BF)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    clean = vpq.ops.paged_attention(q, c, table, dl)
    c.v[table[1, 2].long(), 0, 3, 7] = float("inf")      # token 35 of sequence 1
    q[2, 1, 5] = float("nan")
    got = vpq.ops.paged_attention(q, c, table, dl)
    assert torch.equal(got[0], clean[0])
    assert not got[1, :, 7].isfinite().any() and torch.equal(got[1, :, :7], clean[1, :, :7])
    assert got[2, 1].isnan().all() and torch.equal(got[2, [0, 2, 3]], clean[2, [0, 2, 3]])


@pytest.mark.parametrize("room", [0, 600])
@pytest.mark.parametrize("per", [4, 7, 12])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_8_bits_nan_and_infinity_stay_with_their_group(vpq, D, per, room):
    """64 values with a NaN or an infinity among them are NaN as a whole; the other groups of the row, the other heads
    and the other sequences are what they would be without. (`room`: more columns of the table, so both splits.)"""
    g = gen(14 + D)
    lens, ps, G = [40, 50, 700, 90], 16, D // 64
    c, table = filled(vpq, g, "dense", lens, ps, 2, D, 8)
    wide = torch.nn.functional.pad(table, (0, room), value=1 << 30)
    q = normal(g, 4, 2 * per, D).to(BF)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    clean = vpq.ops.paged_attention(q, c, wide, dl)
    want, tol = ref_attention(q, c, table, lens, 1 / math.sqrt(D), 0)
    at = lambda b, t: (table[b, t // ps].long(), slice(None), t % ps)  # noqa: E731
    # (sequence, token, key head, group): the first token, one in the middle and the last
    spoilt = [(1, 35, 0, G - 1), (2, 0, 1, 0), (2, 350, 1, 0), (2, 699, 1, 0)]
    bad = torch.zeros(4, 2, G, dtype=torch.bool, device="cuda")
    for i, (b, t, h, grp) in enumerate(spoilt):
        page, _, place = at(b, t)
        c.v_scales[page, h, place, grp] = float("nan")  # what the store makes of such a group
        if i == 2:
            c.v_scales[page, h, place, grp] = torch.tensor([float("inf"), 0.0], dtype=BF, device="cuda")  # another's pages
        bad[b, h, grp] = True
    page, _, place = at(3, 17)
    c.k_scales[page, 0, place, 0] = float("nan")  # a key: every weight of its head is NaN
    bad[3, 0] = True
    got = vpq.ops.paged_attention(q, c, wide, dl)
    dead = bad.repeat_interleave(per, 1).repeat_interleave(64, 2)
    assert not got[dead].isfinite().any()
    err = (got.to(F64) - want).abs()
    assert (err <= tol)[~dead].all(), float((err / tol)[~dead].max())
    same = (~bad.any(2)).repeat_interleave(per, 1)
    assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_bad_pages_and_lengths(vpq, bits):
    g = gen(15)
    lens = [40, 64, 20]
    c, table = filled(vpq, g, "dense", lens, 16, 2, 64, bits)
    q = normal(g, 3, 4, 64).to(BF)
    # a page outside holds no tokens
    bad = table.clone()
    bad[0, 1], bad[1, :4] = c.num_pages, -1
    got = vpq.ops.paged_attention(q, c, bad, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert indexes_reported(vpq) == 1
    assert (got[1] == 0).all()
    keep = torch.cat([torch.arange(16), torch.arange(32, 40)]).to("cuda")
    k, v = (at_slots(x, table[0, keep // 16].long() * 16 + keep % 16, 16) for x in held(c))
    for h in range(2):
        p = torch.softmax(q[0, 2 * h:2 * h + 2].to(F64) @ k[:, h].T / 8, -1)
        want, size = p @ v[:, h], p @ v[:, h].abs().amax(-1, keepdim=True)
        assert ((got[0, 2 * h:2 * h + 2].to(F64) - want).abs() <= U * want.abs() + 3 * U * size).all()
    # a length past the table is cut to it; a negative one is an empty sequence
    cut = table[:, :2].contiguous()
    got = vpq.ops.paged_attention(q, c, cut, torch.tensor([2000000000, 33, -4], dtype=torch.int32, device="cuda"))
    assert indexes_reported(vpq) == 8
    want, tol = ref_attention(q, c, cut, [32, 32, 0], 1 / 8, 0)
    assert ((got.to(F64) - want).abs() <= tol).all()


def test_attention_strided_queries_and_outputs(vpq):
    g = gen(17)
    lens = [70, 0, 130]
    c, table = filled(vpq, g, "dense", lens, 16, 2, 64, 16)
    rows = normal(g, 3, 12, 64).to(BF)
    outs = torch.full((3, 20, 64), 5.0, dtype=BF, device="cuda")
    want = check_attention(vpq, rows[:, 2:10].contiguous(), c, table, lens)
    got = vpq.ops.paged_attention(rows[:, 2:10], c, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), out=outs[:, 4:12])
    assert torch.equal(got, want)
    assert (outs[:, :4] == 5).all() and (outs[:, 12:] == 5).all()


def test_attention_after_a_refused_call_and_with_the_widest_window(vpq):
    """A refused call leaves nothing behind that a later one trips over; a window may be as wide as its type."""
    g = gen(19)
    lens = [70, 700]
    c, table = filled(vpq, g, "dense", lens, 16, 2, 64, 16)
    q = normal(g, 2, 8, 64).to(BF)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    with pytest.raises(vpq.VpqError):
        vpq.ops.paged_attention(q, c, table[:, :0], dl)
    for window in (0, 2 ** 31 - 1, 2 ** 31 - 16):
        check_attention(vpq, q, c, table, lens, window=window)
    with pytest.raises(ValueError, match="one page"):
        vpq.ops.PagedKVCache.empty(0, 16, 2, 64)
    for window in (-1, 2 ** 31, 2 ** 32 + 5):
        with pytest.raises(ValueError, match="window"):
            vpq.ops.paged_attention(q, c, table, dl, window=window)


def test_attention_slices_of_tables_and_single_pages(vpq):
    """A page table that is part of a wider one; a cache of one page and one head whose other strides mean nothing."""
    g = gen(18)
    lens = [70, 33, 130]
    c, table = filled(vpq, g, "dense", lens, 16, 2, 64, 16)
    q = normal(g, 3, 8, 64).to(BF)
    want = check_attention(vpq, q, c, table, lens)
    wide = torch.full((5, table.shape[1] + 7), -1, dtype=torch.int32, device="cuda")
    wide[1:4, 3:3 + table.shape[1]] = table
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    assert torch.equal(vpq.ops.paged_attention(q, c, wide[1:4, 3:3 + table.shape[1]], dl), want)
    for bits in (16, 8):
        one = vpq.ops.PagedKVCache.empty(1, 48, 1, 64, bits)
        odd = [None if t is None else torch.as_strided(t, t.shape, (1, 3) + t.stride()[2:]) for t in (one.k, one.v, one.k_scales, one.v_scales)]
        two = vpq.ops.PagedKVCache(*odd)
        x = normal(g, 40, 1, 64).to(BF)
        slots = torch.arange(40, device="cuda")
        vpq.ops.kv_store(x, x, two, slots)
        for a, b in zip(vpq.ops.kv_load(one, slots), vpq.ops.kv_load(two, slots)):
            assert torch.equal(a, b)
        check_attention(vpq, q[:1, :4], two, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), [40])
    with pytest.raises(ValueError, match="page_table"):
        vpq.ops.paged_attention(q, c, table.t().contiguous().t(), dl)


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_in_a_graph_follows_the_lengths(vpq, bits):
    """Captured once, replayed for other lengths, queries and page tables; two graphs on two streams at once."""
    g = gen(19)
    lens = [50, 300, 1]
    c, table = filled(vpq, g, "dense", [400, 400, 400], 16, 2, 128, bits)
    made = []
    for i in range(2):
        q = normal(g, 3, 8, 128).to(BF)
        dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        vpq.ops.paged_attention(q, c, table, dl)
        torch.cuda.synchronize()
        graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=s):
            out = vpq.ops.paged_attention(q, c, table, dl)
        made.append((graph, q, dl, out, s))
    for step, now in enumerate(([0, 400, 17], [399, 2, 0], [128, 128, 128])):
        for graph, q, dl, out, s in made:
            q.copy_(normal(g, 3, 8, 128))
            dl.copy_(torch.tensor(now, dtype=torch.int32))
        torch.cuda.synchronize()
        for graph, q, dl, out, s in made:
            with torch.cuda.stream(s):
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for graph, q, dl, out, s in made:
            assert torch.equal(out, vpq.ops.paged_attention(q, c, table, dl)), (step, now)


def test_first_calls_of_a_process_may_be_captured():
    """What a call looks up once per device (kernels, the status word) may be looked up while a graph is captured."""
    import os
    import subprocess
    import sys
    code = """
import torch, vpipe_b200
ops = vpipe_b200.ops
c = ops.PagedKVCache.empty(8, 16, 2, 64, 8)
q, k = torch.randn(1, 4, 64, device="cuda").bfloat16(), torch.randn(1, 2, 64, device="cuda").bfloat16()
slot, lens = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
table = torch.zeros(1, 8, dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a, b = ops.qk_norm_rope(q, k)
    ops.kv_store(k, k, c, slot)
    o = ops.paged_attention(a, c, table, lens)
    x, _ = ops.kv_load(c, slot)
slot.fill_(999)
g.replay()
torch.cuda.synchronize()
try:
    ops.device_status()
except vpipe_b200.VpqError as e:
    assert e.status == 8
else:
    raise AssertionError("a slot outside was not reported")
slot.fill_(5)
lens.fill_(6)
g.replay()
torch.cuda.synchronize()
assert ops.device_status() == 0 and torch.equal(a, q)
assert (x.float() - k.float()).abs().max() < 0.02
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("hkv", [8, 1])
def test_attention_workspace_contents_do_not_matter(vpq, hkv):
    """The workspace needs no initialisation: whatever is in it, also what the call before left there, the result is
    the same, call after call."""
    import ctypes as C

    from vpipe_b200 import _lib
    g = gen(20)
    lens = [3000, 0, 777, 20011]
    c, table = filled(vpq, g, "dense", lens, 16, hkv, 128, 16)
    q = normal(g, len(lens), 4 * hkv, 128).to(BF)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = check_attention(vpq, q, c, table, lens)
    out = torch.empty_like(want)
    d = _lib.PagedAttentionDesc(q.data_ptr(), out.data_ptr(), 0, 0, table.data_ptr(), dl.data_ptr(), 0, len(lens),
                                table.shape[1], q.shape[1], 0, 0.0)
    L = vpq.lib()
    need = L.vpq_paged_attention_bytes(C.byref(d), c.ref)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    for fill in (0, 255, None, None, 1, "random", None, None):
        if fill == "random":
            ws.copy_(torch.randint(0, 256, (need,), generator=g, device="cuda", dtype=torch.uint8))
        elif fill is not None:
            ws.fill_(fill)
        out.fill_(float("nan"))
        assert L.vpq_paged_attention_bf16(C.byref(d), c.ref, ws.data_ptr(), need, st) == 0
        assert torch.equal(out, want), fill


def test_attention_repeats_itself(vpq):
    """Hundreds of calls and replays over uneven batches, all CTAs of a call meeting in the joins: bit for bit the same."""
    g = gen(22)
    for trial in range(6):
        B = [1, 3, 40, 200, 7, 64][trial]
        lens = (torch.rand(B, generator=g, device="cuda") ** 3 * 3000).int()
        lens[0] = 2999
        c, table = filled(vpq, g, "dense", [3000], 16, [8, 2, 8, 4, 16, 3][trial], 64, 8 if trial % 2 else 16)
        table = table.expand(B, -1).contiguous()
        q = normal(g, B, 2 * c.kv_heads, 64).to(BF)
        want = vpq.ops.paged_attention(q, c, table, lens)
        ref, tol = ref_attention(q, c, table, lens.tolist(), 1 / 8, 0)
        assert ((want.to(F64) - ref).abs() <= tol).all()
        bad = torch.zeros((), dtype=torch.bool, device="cuda")
        for _ in range(60):
            bad |= (vpq.ops.paged_attention(q, c, table, lens) != want).any()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [vpq.ops.paged_attention(q, c, table, lens) for _ in range(4)]
        for _ in range(40):
            for o in outs:
                o.fill_(float("nan"))
            graph.replay()
            for o in outs:
                bad |= (o != want).any()
        assert not bad.item(), trial


def test_calls_on_another_stream(vpq):
    g = gen(21)
    lens = [500, 20]
    c, table = filled(vpq, g, "dense", lens, 16, 2, 128, 8)
    q = normal(g, 2, 8, 128).to(BF)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = vpq.ops.paged_attention(q, c, table, dl)
    slots = torch.arange(16, device="cuda")
    wk, wv = vpq.ops.kv_load(c, slots)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = [vpq.ops.paged_attention(q, c, table, dl, stream=s) for _ in range(20)]
    k, v = vpq.ops.kv_load(c, slots, stream=s)
    s.synchronize()
    assert all(torch.equal(x, want) for x in got) and torch.equal(k, wk) and torch.equal(v, wv)


@pytest.mark.parametrize("bits", [16, 8])
def test_a_cache_beyond_32_bit_offsets(vpq, bits):
    """Pages whose byte offsets (and, for codes, element offsets) pass 2^32; only those are touched."""
    ps, heads, D = 64, 8, 128
    per = heads * ps * D * (bits // 8)
    pages = (1 << 32) // per + 40
    c = vpq.ops.PagedKVCache.empty(pages, ps, heads, D, bits)
    g = gen(23)
    lens = [1000, 333]
    table = torch.stack([torch.arange(pages - 20, pages - 4), torch.arange(pages - 36, pages - 20)]).int().cuda()
    table[0, 0] = pages - 1
    ks, sl = [], []
    for b, n in enumerate(lens):
        t = torch.arange(n, device="cuda")
        sl.append(table[b, t // ps].long() * ps + t % ps)
        ks.append([(normal(g, n, heads, D)).to(BF) for _ in range(2)])
        vpq.ops.kv_store(*ks[b], c, sl[b])
    assert int(sl[0].max()) * heads * D * (bits // 8) > 1 << 32
    small = vpq.ops.PagedKVCache.empty(40, ps, heads, D, bits)
    for b in range(2):
        vpq.ops.kv_store(*ks[b], small, sl[b] - (pages - 40) * ps)
        for x, y in zip(vpq.ops.kv_load(c, sl[b]), vpq.ops.kv_load(small, sl[b] - (pages - 40) * ps)):
            assert torch.equal(x, y)
    q = normal(g, 2, 32, D).to(BF)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    assert torch.equal(vpq.ops.paged_attention(q, c, table, dl),
                       vpq.ops.paged_attention(q, small, table - (pages - 40), dl))


# ------------------------------------------------------------------------------------- as they are used
@pytest.mark.parametrize("bits", [16, 8])
def test_decode_steps_from_projection_to_projection(vpq, oracle_mod, bits):
    """A prompt into the cache, then steps of one token for three users: norm + q|k|v GEMV, norm + rotation + store,
    attention, o GEMV + residual, every launch on one stream without a wait; against a dense 64-bit attention over
    what the q|k|v GEMVs gave."""
    from test_gpu_parity import quantized_linear, to_dev
    g = gen(31)
    hidden, hq, hkv, D, ps, users, steps = 512, 8, 2, 64, 16, 3, 4
    width = (hq + 2 * hkv) * D
    wq = [to_dev(t, dt) for t, dt in zip(quantized_linear(oracle_mod, width, hidden, 1), (None, BF, BF))]
    wo = [to_dev(t, dt) for t, dt in zip(quantized_linear(oracle_mod, hidden, hq * D, 2), (None, BF, BF))]
    qw, kw = (1 + 0.1 * normal(g, D)).to(BF), (1 + 0.1 * normal(g, D)).to(BF)
    table = angles(200, D, g)
    c = vpq.ops.PagedKVCache.empty(30, ps, hkv, D, bits)
    pt = torch.randperm(30, generator=g, device="cuda").int().view(3, 10)
    start = [37, 1, 90]
    hist_k, hist_v = [[] for _ in range(users)], [[] for _ in range(users)]
    slot = lambda b, t: pt[b, t // ps].long() * ps + t % ps  # noqa: E731
    for b in range(users):  # prompts
        n = start[b]
        q, k, v = (normal(g, n, h, D).to(BF) for h in (hq, hkv, hkv))
        pos = torch.arange(n, device="cuda", dtype=torch.int32)
        vpq.ops.qkv_norm_rope_store(q, k, v, qw, kw, table, pos, c, slot(b, pos.long()))
        hist_k[b].append(ref_norm_rope(k, kw, table, pos.long(), 1e-6, False)[0])
        hist_v[b].append(v.to(F64))
    for step in range(steps):
        x = normal(g, users, hidden).to(BF)
        at = torch.tensor([n + step for n in start], device="cuda")
        slots = torch.stack([slot(b, at[b]) for b in range(users)])
        rows = vpq.ops.qmv(*wq, x).view(users, hq + 2 * hkv, D)
        q, k, v = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:]
        qo = vpq.ops.qkv_norm_rope_store(q, k, v, qw, kw, table, at.int(), c, slots)
        o = vpq.ops.paged_attention(qo, c, pt, (at + 1).int())
        y = vpq.ops.qmv_add(*wo, o.view(users, hq * D), x)
        plain = vpq.ops.qmv(*wo, o.view(users, hq * D))
        assert torch.equal(y, (plain.float() + x.float()).to(BF))
        rq = ref_norm_rope(q, qw, table, at, 1e-6, False)[0]
        rk = ref_norm_rope(k, kw, table, at, 1e-6, False)[0]
        for b in range(users):
            hist_k[b].append(rk[b:b + 1])
            hist_v[b].append(v[b:b + 1].to(F64))
            kk, vv = torch.cat(hist_k[b]), torch.cat(hist_v[b])
            for h in range(hkv):
                qq = rq[b, h * 4:(h + 1) * 4]
                s = qq @ kk[:, h].T / 8
                p = torch.softmax(s, -1)
                want = p @ vv[:, h]
                # q and k rounded (bf16, or half a code step of at most spread / 255 with the scale's rounding up), so
                # every score moves by at most ds and every weight by 2 ds relative; then v's and p's rounding
                kerr = U * kk[:, h].abs() if bits == 16 else (kk[:, h].amax(-1, keepdim=True) - kk[:, h].amin(-1, keepdim=True)) / 505
                verr = 0 * vv[:, h] if bits == 16 else ((vv[:, h].amax(-1, keepdim=True) - vv[:, h].amin(-1, keepdim=True)) / 505).expand_as(vv[:, h])
                ds = float(((U * qq.abs()) @ kk[:, h].abs().T + qq.abs() @ kerr.expand_as(kk[:, h]).T).max()) / 8 * 1.02
                size = p @ vv[:, h].abs()
                tol = U * want.abs() + math.expm1(2 * ds) * size * 1.02 + (2 * U if bits == 16 else 4 * H) * (p @ vv[:, h].abs().amax(-1, keepdim=True)) + 1.05 * (p @ verr) * math.exp(2 * ds)
                assert ((o[b, h * 4:(h + 1) * 4].to(F64) - want).abs() <= tol).all()
