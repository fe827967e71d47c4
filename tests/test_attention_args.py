"""CPU tests of the attention block's entry points: what they refuse, with which status, before any launch; and how
the Python front end refuses. Valid calls end at VPQ_ERR_CUDA here (no CPU path)."""
import ctypes as C

import pytest
import torch

from vpipe_b200 import _lib

INVALID, ALIGN, UNSUPPORTED, CUDA = 1, 2, 3, 4
P = 0x7F0000000000  # an address that is never used: every call below ends on the host

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses below are made up: host checks only")


def cache(**kw):
    c = _lib.KvCache()
    c.k, c.v, c.num_pages, c.page_size, c.kv_heads, c.head_dim, c.bits = P, P + (1 << 30), 64, 32, 8, 128, 16
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def cache8(**kw):
    return cache(**{**dict(bits=8, k_scales=P + (2 << 30), v_scales=P + (3 << 30)), **kw})


def qk(**kw):
    d = _lib.QkDesc()
    d.q, d.k, d.v, d.q_out, d.k_out = P, P + 4096, P + 8192, P + 16384, P + 32768
    d.M, d.q_heads, d.kv_heads, d.head_dim, d.eps = 3, 32, 8, 128, 1e-6
    d.cos_sin, d.positions, d.table_rows, d.rot_dim = P + 65536, P + 131072, 100, 128
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def attn(**kw):
    d = _lib.PagedAttentionDesc()
    d.q, d.out, d.page_table, d.seq_lens = P, P + 4096, P + 8192, P + 16384
    d.batch, d.max_pages, d.q_heads = 4, 10, 32
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def norm_rope(L, d):
    return L.vpq_qk_norm_rope_bf16(C.byref(d), None)


def store_pass(L, d, c, slots=P):
    return L.vpq_qkv_norm_rope_store_bf16(C.byref(d), C.byref(c), slots, None)


def attend(L, d, c, ws=P, size=1 << 30):
    return L.vpq_paged_attention_bf16(C.byref(d), C.byref(c), ws, size, None)


def test_valid_calls_reach_the_device_check(vpq):
    L = vpq.lib()
    assert norm_rope(L, qk()) == CUDA
    assert norm_rope(L, qk(q_out=P, k_out=P + 4096)) == CUDA
    assert norm_rope(L, qk(cos_sin=None, positions=None, rot_dim=0, table_rows=0)) == CUDA
    assert norm_rope(L, qk(positions=None)) == CUDA
    for c in (cache(), cache8(), cache(page_stride=128 * 8 * 32 * 2, head_stride=128, token_stride=1024)):
        assert store_pass(L, qk(), c) == CUDA
        assert L.vpq_kv_store_bf16(C.byref(c), P, P, 0, 0, P, 5, None) == CUDA
        assert L.vpq_kv_load_bf16(C.byref(c), P, P, 0, 2048, P, 5, None) == CUDA
        assert attend(L, attn(), c) == CUDA


@pytest.mark.parametrize("kw,code", [
    (dict(M=0), INVALID), (dict(M=-1), INVALID), (dict(q_heads=0), INVALID), (dict(kv_heads=0), INVALID),
    (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED), (dict(q=None), INVALID), (dict(k=None), INVALID),
    (dict(q_out=None), INVALID), (dict(k_out=None), INVALID), (dict(q=P + 8), ALIGN), (dict(k=P + 2), ALIGN),
    (dict(q_out=P + 4), ALIGN), (dict(q_stride=4095), INVALID), (dict(q_stride=4100), ALIGN),
    (dict(k_stride=1000), INVALID), (dict(k_stride=-1024), INVALID), (dict(q_stride=1 << 62), INVALID),
    (dict(rot_dim=8), INVALID), (dict(rot_dim=144), INVALID), (dict(rot_dim=0), INVALID), (dict(rot_dim=-16), INVALID),
    (dict(table_rows=0), INVALID), (dict(positions=None, table_rows=2), INVALID), (dict(positions=P + 2), ALIGN),
    (dict(cos_sin=P + 4), ALIGN), (dict(cos_sin=None), INVALID), (dict(cos_sin=None, rot_dim=0), INVALID),
    (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(q_norm_w=P + 2), ALIGN),
    (dict(k_norm_w=P + 8), ALIGN), (dict(q_out=P, q_out_stride=8192), INVALID),
    (dict(k_out=P + 4096, k_out_stride=2048), INVALID), (dict(q_heads=1 << 20), UNSUPPORTED),
])
def test_norm_rope_refuses(vpq, kw, code):
    assert norm_rope(vpq.lib(), qk(**kw)) == code
    assert vpq.lib().vpq_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(bits=4), UNSUPPORTED), (dict(bits=8), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID),
    (dict(num_pages=0), INVALID), (dict(num_pages=1 << 31), INVALID), (dict(kv_heads=0), INVALID),
    (dict(head_dim=80), UNSUPPORTED), (dict(page_size=0), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED),
    (dict(page_size=-16), UNSUPPORTED), (dict(k=P + 8), ALIGN), (dict(v=P + 1), ALIGN), (dict(k_scales=P), INVALID),
    (dict(token_stride=64, head_stride=4096, page_stride=32768), INVALID),
    (dict(token_stride=132, head_stride=8192, page_stride=65536), ALIGN),
    (dict(token_stride=128, head_stride=0, page_stride=32768), INVALID),
    (dict(token_stride=128, head_stride=4096, page_stride=-32768), INVALID),
    (dict(token_stride=128, head_stride=4096, page_stride=1 << 60), INVALID),
    (dict(token_stride=1 << 30, head_stride=4096, page_stride=32768), INVALID),
    (dict(token_stride=128, head_stride=1 << 30, page_stride=32768), INVALID),
])
def test_a_cache_is_checked(vpq, kw, code):
    L = vpq.lib()
    c = cache(**kw)
    assert L.vpq_kv_store_bf16(C.byref(c), P, P, 0, 0, P, 5, None) == code
    assert L.vpq_kv_load_bf16(C.byref(c), P, P, 0, 0, P, 5, None) == code
    heads = 32 if c.kv_heads <= 0 else 4 * c.kv_heads
    assert attend(L, attn(q_heads=heads), c) == code


@pytest.mark.parametrize("kw,code", [
    (dict(k_scales=None), INVALID), (dict(v_scales=None), INVALID), (dict(k_scales=P + 4), ALIGN),
    (dict(scale_token_stride=2, scale_head_stride=128, scale_page_stride=1024), INVALID),
    (dict(scale_token_stride=6, scale_head_stride=192, scale_page_stride=1536), ALIGN),
    (dict(token_stride=136, head_stride=8192, page_stride=65536), ALIGN),
])
def test_an_8_bit_cache_is_checked(vpq, kw, code):
    L = vpq.lib()
    c = cache8(**kw)
    assert L.vpq_kv_store_bf16(C.byref(c), P, P, 0, 0, P, 5, None) == code
    assert attend(L, attn(), c) == code


def test_an_8_bit_cache_with_scale_strides_out_of_range_is_refused(vpq):
    """The pairs of up to four heads are addressed with 32 bits, so a scale's strides, two bytes an element, end where those
    of bf16 pages do: below 2^30 bytes."""
    L = vpq.lib()
    far, last = 1 << 29, (1 << 29) - 4  # elements of two bytes

    def calls(c):
        yield L.vpq_kv_store_bf16(C.byref(c), P, P, 0, 0, P, 5, None)
        yield L.vpq_kv_load_bf16(C.byref(c), P, P, 0, 0, P, 5, None)
        yield store_pass(L, qk(), c)
        yield attend(L, attn(), c)

    for token, head in ((4, far), (far, 128), (4, far + 1024), (4, (1 << 30) - 4), ((1 << 30) - 4, 128)):
        c = cache8(scale_token_stride=token, scale_head_stride=head, scale_page_stride=1 << 33)
        assert set(calls(c)) == {INVALID}, (token, head)
    for token, head in ((4, last), (last, 128)):
        c = cache8(scale_token_stride=token, scale_head_stride=head, scale_page_stride=1 << 33)
        assert set(calls(c)) == {CUDA}, (token, head)


def test_store_pass_refuses(vpq):
    L = vpq.lib()
    assert store_pass(L, qk(v=None), cache()) == INVALID
    assert store_pass(L, qk(v=P + 2), cache()) == ALIGN
    assert store_pass(L, qk(v_stride=100), cache()) == INVALID
    assert store_pass(L, qk(), cache(kv_heads=4)) == INVALID
    assert store_pass(L, qk(), cache(head_dim=64)) == INVALID
    assert store_pass(L, qk(), cache(), None) == INVALID
    assert store_pass(L, qk(), cache(), P + 4) == ALIGN
    assert L.vpq_qkv_norm_rope_store_bf16(None, C.byref(cache()), P, None) == INVALID
    assert L.vpq_qkv_norm_rope_store_bf16(C.byref(qk()), None, P, None) == INVALID
    assert L.vpq_qk_norm_rope_bf16(None, None) == INVALID


def test_store_and_load_refuse(vpq):
    L = vpq.lib()
    for f in (L.vpq_kv_store_bf16, L.vpq_kv_load_bf16):
        c = C.byref(cache())
        assert f(None, P, P, 0, 0, P, 5, None) == INVALID
        assert f(c, None, P, 0, 0, P, 5, None) == INVALID
        assert f(c, P, None, 0, 0, P, 5, None) == INVALID
        assert f(c, P, P, 0, 0, None, 5, None) == INVALID
        assert f(c, P, P, 0, 0, P, 0, None) == INVALID
        assert f(c, P, P, 0, 0, P, -3, None) == INVALID
        assert f(c, P, P, 512, 0, P, 5, None) == INVALID
        assert f(c, P, P, 0, 1028, P, 5, None) == ALIGN
        assert f(c, P + 2, P, 0, 0, P, 5, None) == ALIGN
        assert f(c, P, P, 0, 0, P + 2, 5, None) == ALIGN


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(page_table=None), INVALID), (dict(seq_lens=None), INVALID),
    (dict(batch=0), INVALID), (dict(batch=-2), INVALID), (dict(max_pages=0), INVALID), (dict(q_heads=0), INVALID),
    (dict(q_heads=12), INVALID), (dict(q_heads=65544), UNSUPPORTED), (dict(window=-1), INVALID),
    (dict(scale=-0.5), INVALID), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
    (dict(q=P + 2), ALIGN), (dict(out=P + 8), ALIGN), (dict(q_stride=4092), INVALID), (dict(q_stride=4100), ALIGN),
    (dict(out_stride=100), INVALID), (dict(out_stride=1 << 50), INVALID), (dict(table_stride=9), INVALID),
    (dict(page_table=P + 2), ALIGN), (dict(seq_lens=P + 1), ALIGN), (dict(max_pages=1 << 27), UNSUPPORTED),
])
def test_paged_attention_refuses(vpq, kw, code):
    assert attend(vpq.lib(), attn(**kw), cache()) == code
    assert vpq.lib().vpq_last_error()


# f32 numbers around the ends of what a scale may be: 2^-126, and the largest whose product with log2(e) is a number.
SMALLEST, LARGEST = 2.0 ** -126, 2.3586e38


@pytest.mark.parametrize("scale,code", [
    (2.0 ** -149, INVALID), (1e-40, INVALID), (1.17e-38, INVALID), (2.37e38, INVALID), (3.3e38, INVALID), (3.4e38, INVALID),
    (SMALLEST, CUDA), (1e-30, CUDA), (1.0, CUDA), (2.35e38, CUDA), (LARGEST, CUDA), (0.0, CUDA),
])
def test_paged_attention_scales_at_the_ends_of_their_range(vpq, scale, code):
    """A scale below the normal numbers, or one whose product with log2(e) is not a number, does not weigh as it says."""
    for c in (cache(), cache8()):
        assert attend(vpq.lib(), attn(scale=scale), c) == code


def test_python_refuses_scales_that_f32_does_not_hold(vpq):
    """1e-46 is positive and becomes 0 in f32, which means 1 / sqrt(head_dim) to the library."""
    for scale in (1e-46, 1e-300, 1e-40, 0.0, -1.0, 2.37e38, 1e39, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            vpq.ops._scale(scale)
    for scale in (SMALLEST, 1e-30, 0.125, 1, LARGEST):
        assert vpq.ops._scale(scale) == scale
    assert vpq.ops._scale(None) == 0.0


def test_paged_attention_workspace(vpq):
    L = vpq.lib()
    need = L.vpq_paged_attention_bytes(C.byref(attn()), C.byref(cache()))
    assert need > 0
    assert attend(L, attn(), cache(), P, need) == CUDA
    assert attend(L, attn(), cache(), P, need - 1) == INVALID
    assert attend(L, attn(), cache(), None, need) == INVALID
    assert attend(L, attn(), cache(), P + 8, need) == ALIGN
    assert L.vpq_paged_attention_bytes(None, C.byref(cache())) == 0
    assert L.vpq_paged_attention_bytes(C.byref(attn(q_heads=12)), C.byref(cache())) == 0
    # any batch: what is kept between the two kernels goes by the CTAs, not by the sequences
    assert L.vpq_paged_attention_bytes(C.byref(attn(batch=1 << 20)), C.byref(cache())) == need


def test_python_refuses_cpu_tensors_and_wrong_types(vpq):
    ops = vpq.ops
    q, k = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.qk_norm_rope(q, k)
    with pytest.raises(ValueError, match="bfloat16"):
        ops.qk_norm_rope(q.float(), k)
    pages = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.PagedKVCache(pages, pages.clone())
    with pytest.raises(ValueError, match="scales"):
        ops.PagedKVCache(pages.to(torch.uint8), pages.to(torch.uint8))
    with pytest.raises(ValueError, match="16 or 8"):
        ops.PagedKVCache.empty(2, 16, 2, 64, bits=4, device="cpu")


def test_packed_descriptors_are_the_structures(vpq):
    for cls, fields in ((_lib.QkDesc, 22), (_lib.PagedAttentionDesc, 12)):
        values = [2 ** 40 + 7 * i if i < 5 else 3 + i for i in range(fields - 1)] + [0.25]
        if cls is _lib.PagedAttentionDesc:
            values[6] = 2 ** 40
        assert bytes(cls(*values)) == cls.pack(*values)


def test_broadcast_rows_are_refused(vpq):
    """Stride 0 means "dense" to the library, so rows that share their memory would be read past its end."""
    rows = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    assert vpq.ops._heads("q", rows, -1, rows.shape)[1] == 0
    with pytest.raises(ValueError, match="share"):
        vpq.ops._heads("q", rows.expand(5, 4, 64), -1, (5, 4, 64))
    one = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16).expand(3, 2, 16, 64)
    with pytest.raises(ValueError, match="share"):
        vpq.ops.PagedKVCache(one, one)
    codes = torch.zeros(3, 2, 16, 64, dtype=torch.uint8)
    pairs = torch.zeros(1, 1, 1, 1, 2, dtype=torch.bfloat16).expand(3, 2, 16, 1, 2)
    with pytest.raises(ValueError, match="share"):
        vpq.ops.PagedKVCache(codes, codes, pairs, pairs)


def test_page_tables_that_may_be_parts_of_wider_ones(vpq):
    t = torch.zeros(6, 9, dtype=torch.int32)
    part = t[1:4, 2:7]
    assert vpq.ops._table(part, -1, 3) == (part.data_ptr(), 9, 5)
    assert vpq.ops._table(t[:1, :4], -1, 1)[1:] == (0, 4)
    assert vpq.ops._table(t[:, 3].unsqueeze(1), -1, 6)[1:] == (9, 1)
    # stride 0 means "dense" to the library: a broadcast table would be read past its end
    for bad in (t[:1, :4].expand(3, 4), t[:, :1].expand(6, 4), t.t(), t[0], t.long(), t[:, ::2]):
        with pytest.raises(ValueError, match="page_table"):
            vpq.ops._table(bad, -1, bad.shape[0])
    with pytest.raises(ValueError, match="page_table"):
        vpq.ops._table(t, -1, 5)


def test_status_string_of_a_bad_index(vpq):
    assert vpq.status_string(8) not in ("ok", "unknown status")
