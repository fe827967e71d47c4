"""The attention block of a decode step and of a prompt, between the q | k | v projection and the output projection:
what it costs, and what it has to give.

Three operators: the per-head norm of queries and keys with the position rotation (alone, or with keys and values going
straight into the paged cache), the paged cache's own store and load (bf16, or 8-bit codes with a scale and a bias
per 64 values), and the attention of one new token per sequence over that cache.

`own` False: the plain form, elementary torch operations in 32 bits. `own` True: the calls a user makes.
"""
import math
import random

import torch

own = False

EPS = 1e-6
THETA = 1e6
GROUP = 64  # values that share a scale and a bias of an 8-bit cache

# The 8B decoder of the benchmark: 32 query heads, 8 key / value heads of 128 (q 4096, k and v 1024 wide).


def listed():
    return [
        # one new token of one user: a step's latency
        dict(name="norm_rope_1_token", op="norm_rope", tokens=1, q_heads=32, kv_heads=8, head_dim=128, rot=128,
             interleaved=False, per_row=False),
        # a prompt of the 8B decoder, as its prefill GEMMs take it
        dict(name="norm_rope_prompt", op="norm_rope", tokens=2048, q_heads=32, kv_heads=8, head_dim=128, rot=128,
             interleaved=False, per_row=False),
        # a quarter of the video model's tokens (hidden 5120): every head its own key, rotation by three axes, so one
        # table row per token, neighbouring values paired
        dict(name="norm_rope_video", op="norm_rope", tokens=16320, q_heads=40, kv_heads=40, head_dim=128, rot=128,
             interleaved=True, per_row=True),
        # one new token into an 8-bit cache
        dict(name="store_pass_1_token_w8", op="store_pass", tokens=1, q_heads=32, kv_heads=8, head_dim=128, rot=128,
             bits=8, page_size=64),
        # a decode step of 129 users into a bf16 cache, two rows of the batch padded; part of each head rotated
        dict(name="store_pass_129_partial", op="store_pass", tokens=129, q_heads=16, kv_heads=2, head_dim=256, rot=64,
             bits=16, page_size=32),
        # a chunk of long prompts into an 8-bit cache
        dict(name="store_pass_prompt_w8", op="store_pass", tokens=8191, q_heads=32, kv_heads=8, head_dim=128, rot=128,
             bits=8, page_size=64),
        # a cache written apart from the projection pass (keys that came from elsewhere) and read back for a prompt
        # that goes on from it
        dict(name="cache_w8_512", op="cache", tokens=512, kv_heads=8, head_dim=128, bits=8, page_size=16),
        dict(name="cache_w8_65536", op="cache", tokens=65536, kv_heads=8, head_dim=128, bits=8, page_size=64),
        # one user at the start of a talk
        dict(name="attend_1_short", op="attend", batch=1, longest=333, even=True, q_heads=32, kv_heads=8, head_dim=128,
             bits=16, page_size=64, window=0),
        # one user with a long document
        dict(name="attend_1_long_w8", op="attend", batch=1, longest=131071, even=True, q_heads=32, kv_heads=8,
             head_dim=128, bits=8, page_size=64, window=0),
        # a serving batch, lengths from one token to long ones
        dict(name="attend_64_ragged", op="attend", batch=64, longest=16384, even=False, q_heads=32, kv_heads=8,
             head_dim=128, bits=16, page_size=16, window=0),
        # a large batch with sliding-window layers and wide heads
        dict(name="attend_200_window_w8", op="attend", batch=200, longest=8192, even=False, q_heads=16, kv_heads=4,
             head_dim=256, bits=8, page_size=32, window=1024),
    ]


HEADS = [(32, 8), (16, 8), (40, 8), (64, 8), (28, 4), (8, 1), (12, 12), (16, 2), (7, 1), (24, 2)]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "store_pass", "cache", "attend", "attend"])
    hq, hkv = rng.choice(HEADS)
    d = rng.choice([64, 128, 128, 256])
    rot = rng.choice([d, d, d // 2, d // 4])
    if op == "norm_rope":
        # at most the video case's values
        t = _log(rng, 1, min(16384, 16320 * 80 * 128 // ((hq + hkv) * d)))
        return dict(op=op, tokens=t, q_heads=hq, kv_heads=hkv, head_dim=d, rot=rot, interleaved=rng.random() < 0.4,
                    per_row=rng.random() < 0.3)
    bits, page = rng.choice([8, 16]), rng.choice([16, 32, 48, 64, 128])
    if op == "store_pass":
        t = _log(rng, 1, min(8191, 8191 * 48 * 128 // ((hq + 2 * hkv) * d)))
        return dict(op=op, tokens=t, q_heads=hq, kv_heads=hkv, head_dim=d, rot=rot, bits=bits, page_size=page)
    if op == "cache":
        t = _log(rng, 1, min(65536, 65536 * 1024 // (hkv * d * (bits // 8))))
        return dict(op=op, tokens=t, kv_heads=hkv, head_dim=d, bits=bits, page_size=page)
    batch = _log(rng, 1, 200)
    # no more than the ragged batch's cache, were every sequence the longest
    longest = _log(rng, 1, max(1, min(131072, 64 * 16384 * 1024 // (batch * hkv * d))))
    return dict(op=op, batch=batch, longest=longest, even=rng.random() < 0.4, q_heads=hq, kv_heads=hkv, head_dim=d,
                bits=bits, page_size=page, window=rng.choice([0, 0, 0, 128, 1000]))


def lengths(case):
    """The sequences' lengths: the same for every seed (their order is not)."""
    n, longest = case["batch"], case["longest"]
    if case["even"]:
        return [longest] * n
    r = random.Random(n * 1000003 + longest)
    return [longest] + [max(0, int(round(math.exp(r.uniform(0.0, math.log(longest + 1)))) - 1)) for _ in range(n - 1)]


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFFFFFF)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _channels(g, heads, d):
    """Key channels are not alike: most near one, a few of them large, each with an offset of its own."""
    wide = 1.0 + 5.0 * (torch.rand(heads, d, generator=g, device="cuda") < 0.03).float()
    return wide, 0.5 * wide * _normal(g, heads, d)


def _table(rows, rot, positions=None):
    """cos | sin of every position, made in 64 bits, kept in 32."""
    p = torch.arange(rows, device="cuda", dtype=torch.float64) if positions is None else positions.double()
    f = THETA ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2 / rot)
    a = p[:, None] * f[None, :]
    return torch.cat([a.cos(), a.sin()], dim=1).float().contiguous()


def _slots(g, tokens, page_size, pages, padded):
    """Consecutive places of pages taken in any order; `padded` rows at the end go nowhere."""
    order = torch.randperm(pages, generator=g, device="cuda")
    t = torch.arange(tokens, device="cuda")
    slots = order[t // page_size] * page_size + t % page_size
    if padded:
        slots[tokens - padded:] = -1
    return slots.long().contiguous()


def _projected(case, g):
    """Rows of q | k | v as one projection leaves them, and views of the three parts."""
    m, hq, hkv, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
    wide, off = _channels(g, hq + 2 * hkv, d)
    rows = (_normal(g, m, hq + 2 * hkv, d) * wide + off).to(torch.bfloat16)
    q, k, v = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:]
    qw = (1.0 + 0.2 * _normal(g, d)).to(torch.bfloat16)
    kw = (1.0 + 0.2 * _normal(g, d)).to(torch.bfloat16)
    return q, k, v, qw, kw


def _pages(case, pages):
    shape = (pages, case["kv_heads"], case["page_size"], case["head_dim"])
    c = {}
    for n in ("k", "v"):
        if case["bits"] == 16:
            c[n] = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
            c[n + "s"] = None
        else:
            c[n] = torch.zeros(shape, dtype=torch.uint8, device="cuda")
            c[n + "s"] = torch.zeros(shape[:3] + (shape[3] // GROUP, 2), dtype=torch.bfloat16, device="cuda")
    return c


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case=case)
    op = case["op"]
    if op in ("norm_rope", "store_pass"):
        m, rot = case["tokens"], case["rot"]
        s["q"], s["k"], s["v"], s["qw"], s["kw"] = _projected(case, g)
        if case.get("per_row"):
            where = torch.rand(m, generator=g, device="cuda") * 200.0
            s["table"], s["positions"] = _table(m, rot, where), None
        else:
            s["table"] = _table(40960, rot)
            if op == "norm_rope":  # one prompt, some way into a talk
                start = int(torch.randint(0, 40960 - m, (1,), generator=g, device="cuda"))
                s["positions"] = torch.arange(start, start + m, device="cuda", dtype=torch.int32)
            else:
                s["positions"] = torch.randint(0, 40960, (m,), generator=g, device="cuda", dtype=torch.int32)
    if op in ("store_pass", "cache"):
        m, ps = case["tokens"], case["page_size"]
        pages = -(-m // ps) + 2
        s.update(cache=_pages(case, pages), slots=_slots(g, m, ps, pages, 2 if m >= 100 else 0))
    if op == "cache":
        wide, off = _channels(g, case["kv_heads"], case["head_dim"])
        s["k"] = (_normal(g, m, case["kv_heads"], case["head_dim"]) * wide + off).to(torch.bfloat16)
        s["v"] = _normal(g, m, case["kv_heads"], case["head_dim"]).to(torch.bfloat16)
    if op == "attend":
        hq, hkv, d, ps = case["q_heads"], case["kv_heads"], case["head_dim"], case["page_size"]
        lens = lengths(case)
        order = torch.randperm(len(lens), generator=g, device="cuda")
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")[order].contiguous()
        per = -(-max(case["longest"], 1) // ps)
        need = (s["lens"].long() + ps - 1) // ps
        pages = int(need.sum()) + 3
        place = torch.randperm(pages, generator=g, device="cuda").int()
        at = torch.cumsum(need, 0) - need
        col = torch.arange(per, device="cuda")
        table = place[torch.clamp(at[:, None] + col[None, :], max=pages - 1)]
        s["page_table"] = torch.where(col[None, :] < need[:, None], table, torch.zeros_like(table)).contiguous()
        s["q"] = (1.5 * _normal(g, len(lens), hq, d)).to(torch.bfloat16)
        s["cache"] = c = _pages(case, pages)
        wide, off = _channels(g, hkv, d)
        for n in ("k", "v"):  # page by page: a large cache in 32 bits would not be small
            step = max(1, (1 << 27) // (hkv * ps * d))
            for a in range(0, pages, step):
                b = min(pages, a + step)
                x = _normal(g, b - a, hkv, ps, d)
                if n == "k":
                    x = 0.5 * (x * wide[None, :, None] + off[None, :, None])
                x = x.to(torch.bfloat16)
                if case["bits"] == 16:
                    c[n][a:b] = x
                else:
                    c[n][a:b], c[n + "s"][a:b] = _quantise(x.float())
        return s


# ------------------------------------------------------------------------------------------------ plain forms
def _bf16_down(x):
    """f32 -> the largest bf16 value that is not above it, as f32."""
    i = x.contiguous().view(torch.int32)
    t = i & -65536
    return torch.where((x < 0) & ((i & 65535) != 0), t + 65536, t).view(torch.float32)


def _bf16_up(x):
    return -_bf16_down(-x)


def _quantise(x):
    """f32 [..., d] -> codes [..., d] and (scale, bias) [..., d / 64, 2]."""
    v = x.reshape(x.shape[:-1] + (x.shape[-1] // GROUP, GROUP))
    bias = _bf16_down(v.amin(-1))
    scale = _bf16_up((v.amax(-1) - bias) / 255.0)
    code = torch.round((v - bias[..., None]) / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None])
    code = code.clamp(0, 255).to(torch.uint8)
    return code.reshape(x.shape), torch.stack([scale, bias], -1).to(torch.bfloat16)


def _values(codes, scales):
    """f32 values that codes stand for."""
    v = codes.float().reshape(codes.shape[:-1] + (codes.shape[-1] // GROUP, GROUP))
    sb = scales.float()
    return (v * sb[..., 0:1] + sb[..., 1:2]).reshape(codes.shape)


def _norm(x, w):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()


def _rotate(x, row, interleaved):
    """x [m, heads, d] f32, row [m, rot] = cos | sin."""
    h = row.shape[1] // 2
    c, s = row[:, None, :h], row[:, None, h:]
    if interleaved:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h:2 * h]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y, x[..., 2 * h:]], -1)


def _write(c, slots, ps, k, v, bits):
    """k, v f32 [m, heads, d] into the pages; rows without a place go nowhere."""
    rows = (slots >= 0).nonzero().squeeze(1)
    page, at = slots[rows] // ps, slots[rows] % ps
    for n, x in (("k", k), ("v", v)):
        if bits == 16:
            c[n][page, :, at] = x[rows].to(torch.bfloat16)
        else:
            c[n][page, :, at], c[n + "s"][page, :, at] = _quantise(x[rows])


def _read(c, slots, ps, bits):
    live = (slots >= 0)[:, None, None]
    page, at = slots.clamp(min=0) // ps, slots.clamp(min=0) % ps
    got = []
    for n in ("k", "v"):
        x = c[n][page, :, at]
        x = x.float() if bits == 16 else _values(x, c[n + "s"][page, :, at])
        got.append(torch.where(live, x, torch.zeros_like(x)).to(torch.bfloat16))
    return got


def _plain_attention(s):
    case, c = s["case"], s["cache"]
    table, lens, q = s["page_table"].long(), s["lens"].long(), s["q"].float()
    b, hq, d = q.shape
    hkv, ps = case["kv_heads"], case["page_size"]
    span = table.shape[1] * ps

    def gathered(n):
        x = c[n][table]  # [b, pages, heads, page, d]
        x = x.float() if case["bits"] == 16 else _values(x, c[n + "s"][table])
        return x.transpose(2, 3).reshape(b, span, hkv, d)

    t = torch.arange(span, device=q.device)[None, :]
    live = t < lens[:, None]
    if case["window"]:
        live &= t >= (lens - case["window"])[:, None]
    score = torch.einsum("bhgd,bthd->bhgt", q.reshape(b, hkv, hq // hkv, d), gathered("k")) / math.sqrt(d)
    score = score.masked_fill(~live[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    v = gathered("v").masked_fill(~live[:, :, None, None], 0.0)
    o = torch.einsum("bhgt,bthd->bhgd", p, v) / torch.where(total > 0, total, torch.ones_like(total))
    return o.reshape(b, hq, d).to(torch.bfloat16)


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "attend":
        return _plain_attention(s)
    if op in ("norm_rope", "store_pass"):
        row = s["table"] if s["positions"] is None else s["table"][s["positions"].long()]
        il = case.get("interleaved", False)
        q, k = _rotate(_norm(s["q"], s["qw"]), row, il), _rotate(_norm(s["k"], s["kw"]), row, il)
        if op == "norm_rope":
            return q.to(torch.bfloat16), k.to(torch.bfloat16)
        _write(s["cache"], s["slots"], case["page_size"], k, s["v"].float(), case["bits"])
        return (q.to(torch.bfloat16), *_read(s["cache"], s["slots"], case["page_size"], case["bits"]))
    _write(s["cache"], s["slots"], case["page_size"], s["k"].float(), s["v"].float(), case["bits"])
    return tuple(_read(s["cache"], s["slots"], case["page_size"], case["bits"]))


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    from vpipe_b200 import ops

    case = s["case"]
    op = case["op"]
    if op == "norm_rope":
        return ops.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["table"], s["positions"], eps=EPS,
                                interleaved=case["interleaved"])
    cache = s.get("handle")
    if cache is None:  # what a program makes once for the pages that it keeps
        c = s["cache"]
        cache = s["handle"] = ops.PagedKVCache(c["k"], c["v"], c["ks"], c["vs"])
    if op == "store_pass":
        q = ops.qkv_norm_rope_store(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["table"], s["positions"], cache,
                                    s["slots"], eps=EPS)
        return (q, *ops.kv_load(cache, s["slots"]))
    if op == "cache":
        ops.kv_store(s["k"], s["v"], cache, s["slots"])
        return ops.kv_load(cache, s["slots"])
    return ops.paged_attention(s["q"], cache, s["page_table"], s["lens"], window=case["window"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ what it has to cost
def work(case):
    op, d = case["op"], case["head_dim"]
    held = {16: 2 * d, 8: d + d // GROUP * 4}  # bytes of one head's row in a cache
    if op == "attend":
        n = sum(min(x, case["window"]) if case["window"] else x for x in lengths(case))
        io = case["batch"] * (2 * case["q_heads"] * d * 2 + 4) + 4 * sum(-(-x // case["page_size"]) for x in lengths(case))
        return dict(bytes=2 * n * case["kv_heads"] * held[case["bits"]] + io, flops=4 * n * case["q_heads"] * d)
    m, kv = case["tokens"], case["kv_heads"]
    if op == "cache":
        dense = 2 * m * kv * d * 2
        return dict(bytes=2 * dense + 4 * m * kv * held[case["bits"]] + 16 * m, flops=2 * m * kv * d * 6)
    hq, table = case["q_heads"], 4 * m * case["rot"] + 4 * m
    if op == "norm_rope":
        return dict(bytes=2 * m * (hq + kv) * d * 2 + table, flops=8 * m * (hq + kv) * d)
    written = 2 * m * kv * held[case["bits"]]
    # rows in, queries out, the cache's rows out and in again, their values out
    return dict(bytes=m * (2 * hq + 4 * kv) * d * 2 + table + 2 * written + 16 * m, flops=12 * m * (hq + 2 * kv) * d)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _toward(x, up):
    """f64 -> the nearest bf16 on one side, as f64."""
    b = x.to(torch.bfloat16)
    far = torch.full_like(b, math.inf if up else -math.inf)
    wrong = b.double() < x if up else b.double() > x
    return torch.where(wrong, torch.nextafter(b, far), b).double()


def _held(x, bits):
    """What a cache gives back for x f64 [m, heads, d]; a bf16 one is off by its rounding alone."""
    if bits == 16:
        return x
    parts = []
    for a in range(0, x.shape[-1], GROUP):
        y = x[..., a:a + GROUP]
        lo = _toward(y.min(-1, keepdim=True).values, False)
        step = _toward((y.max(-1, keepdim=True).values - lo) / 255, True)
        n = ((y - lo) / torch.where(step == 0, 1.0, step)).round().clamp(0, 255)
        parts.append(lo + n * step)
    return torch.cat(parts, -1)


def _turned(x, w, cos, sin, interleaved):
    x = x.double()
    x = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
    h = cos.shape[-1]
    z = torch.polar(torch.ones_like(cos), torch.atan2(sin, cos)) * torch.sqrt(cos * cos + sin * sin)
    if interleaved:
        y = torch.view_as_real(torch.view_as_complex(x[..., :2 * h].reshape(*x.shape[:-1], h, 2).contiguous()) * z)
        y = y.reshape(*x.shape[:-1], 2 * h)
    else:
        t = torch.complex(x[..., :h].contiguous(), x[..., h:2 * h].contiguous()) * z
        y = torch.cat([t.real, t.imag], -1)
    return torch.cat([y, x[..., 2 * h:]], -1)


def exact(case, seed):
    s = prepare(case, seed)
    op, bits = case["op"], case.get("bits")
    if op == "attend":
        c, ps, hkv, d = s["cache"], case["page_size"], case["kv_heads"], case["head_dim"]
        per = case["q_heads"] // hkv
        out = torch.zeros(case["batch"], case["q_heads"], d, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens"].tolist()):
            first = max(0, n - case["window"]) if case["window"] else 0
            if n <= first:
                continue
            page = s["page_table"][b, : -(-n // ps)].long()
            for h in range(hkv):
                kv = []
                for name in ("k", "v"):
                    x = c[name][page, h].double().reshape(-1, d)
                    if bits == 8:
                        sb = c[name + "s"][page, h].double().reshape(-1, d // GROUP, 2).repeat_interleave(GROUP, 1)
                        x = x * sb[..., 0] + sb[..., 1]
                    kv.append(x[first:n])
                a = s["q"][b, h * per:(h + 1) * per].double() @ kv[0].T / d ** 0.5
                out[b, h * per:(h + 1) * per] = torch.softmax(a, -1) @ kv[1]
        return out
    live = None if op == "norm_rope" else (s["slots"] >= 0)[:, None, None].double()
    if op == "cache":
        return tuple(_held(s[n].double(), bits) * live for n in ("k", "v"))
    row = (s["table"] if s["positions"] is None else s["table"][s["positions"].long()]).double()
    cos, sin = row[:, None, : case["rot"] // 2], row[:, None, case["rot"] // 2:]
    il = case.get("interleaved", False)
    q, k = _turned(s["q"], s["qw"], cos, sin, il), _turned(s["k"], s["kw"], cos, sin, il)
    if op == "norm_rope":
        return q, k
    return q, _held(k, bits) * live, _held(s["v"].double(), bits) * live
