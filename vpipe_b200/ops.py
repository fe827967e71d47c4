"""Torch-tensor front end to the C ABI (device pointers pass straight through).

16-bit float tensors may be torch.bfloat16 / torch.float16 or raw int16/uint16
bit patterns; packed weights are int32 / uint32 [N, K/8].
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import check, lib


def _ptr(t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise ValueError("vpipe_b200.ops: tensors must live on a CUDA device (no CPU path)")
    if not t.is_contiguous():
        raise ValueError("vpipe_b200.ops: tensors must be contiguous")
    return t.data_ptr()


def _stream(stream=None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def quantize(w: torch.Tensor, clip: float = 1.0, stream=None, bits: int = 4, group: int = 64):
    """Dense [N,K] f16/bf16 -> (codes int32 [N,K*bits/32], scales f16, biases f16 [N,K/group])."""
    if w.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("quantize: w must be float16 or bfloat16")
    N, K = w.shape
    dev = w.device
    with torch.cuda.device(dev):
        codes = torch.empty((N, max(K * bits // 32, 1)), dtype=torch.int32, device=dev)
        s = torch.empty((N, max(K // group, 1)), dtype=torch.float16, device=dev)
        b = torch.empty_like(s)
        if (bits, group) == (4, 64):
            check(lib().vpq_affine_quant_w4_g64(_ptr(w), int(w.dtype == torch.bfloat16), _ptr(codes),
                                                _ptr(s), _ptr(b), K, N, clip, _stream(stream)))
        else:
            check(lib().vpq_affine_quant(_ptr(w), int(w.dtype == torch.bfloat16), _ptr(codes), _ptr(s), _ptr(b),
                                         K, N, bits, group, clip, _stream(stream)))
    return codes, s, b


def dequantize_any(codes, scales, biases, bits: int, group: int, out=None, stream=None) -> torch.Tensor:
    """Any of the format twins (bits 4 | 8, group 64 | 32) -> dense bf16 [N, K]."""
    N, Kw = codes.shape
    K = Kw * 32 // bits
    if out is None:
        out = torch.empty((N, K), dtype=torch.bfloat16, device=codes.device)
    with torch.cuda.device(codes.device):
        check(lib().vpq_affine_dequant_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(out), K, N, bits, group,
                                            _stream(stream)))
    return out


def requant_w8_to_w4(codes8, scales8, biases8, stream=None):
    """8-bit group-64 weights -> (codes int32 [N, K/8], scales bf16, biases bf16 [N, K/64]) at 4 bits
    (vpq_affine_requant_w8_to_w4_g64_bf16)."""
    N, Kw = codes8.shape
    K = Kw * 4
    dev = codes8.device
    codes4 = torch.empty((N, K // 8), dtype=torch.int32, device=dev)
    s4 = torch.empty((N, K // 64), dtype=torch.bfloat16, device=dev)
    b4 = torch.empty((N, K // 64), dtype=torch.bfloat16, device=dev)
    with torch.cuda.device(dev):
        check(lib().vpq_affine_requant_w8_to_w4_g64_bf16(_ptr(codes8), _ptr(scales8), _ptr(biases8), _ptr(codes4),
                                                         _ptr(s4), _ptr(b4), K, N, _stream(stream)))
    return codes4, s4, b4


def narrow_f32_bf16(w: torch.Tensor, stream=None) -> torch.Tensor:
    out = torch.empty(w.shape, dtype=torch.bfloat16, device=w.device)
    with torch.cuda.device(w.device):
        check(lib().vpq_narrow_f32_bf16(_ptr(w), _ptr(out), w.numel(), _stream(stream)))
    return out


def scales_to_bf16(s_f16: torch.Tensor, stream=None) -> torch.Tensor:
    out = torch.empty(s_f16.shape, dtype=torch.bfloat16, device=s_f16.device)
    with torch.cuda.device(s_f16.device):
        check(lib().vpq_scales_f16_to_bf16(_ptr(s_f16), _ptr(out), s_f16.numel(), _stream(stream)))
    return out


def dequantize(codes, scales, biases, out=None, stream=None) -> torch.Tensor:
    N, Kw = codes.shape
    K = Kw * 8
    if out is None:
        out = torch.empty((N, K), dtype=torch.bfloat16, device=codes.device)
    with torch.cuda.device(codes.device):
        check(lib().vpq_affine_dequant_w4g64_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(out),
                                                  K, N, _stream(stream)))
    return out


def qmv(codes, scales, biases, x, out=None, stream=None) -> torch.Tensor:
    N, Kw = codes.shape
    K = Kw * 8
    M = x.numel() // K
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    with torch.cuda.device(x.device):
        check(lib().vpq_affine_qmv_w4g64_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x),
                                              _ptr(out), K, N, M, _stream(stream)))
    return out


def qmv_g32(codes, scales, biases, x, out=None, stream=None) -> torch.Tensor:
    """GEMV over 4-bit group-32 weights, scales / biases [N, K/32] (vpq_affine_qmv_w4g32_bf16)."""
    N, Kw = codes.shape
    K = Kw * 8
    M = x.numel() // K
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    with torch.cuda.device(x.device):
        check(lib().vpq_affine_qmv_w4g32_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x), _ptr(out),
                                              K, N, M, _stream(stream)))
    return out


def qmv_w8(codes, scales, biases, x, out=None, stream=None) -> torch.Tensor:
    """GEMV over 8-bit group-64 weights, codes int32 [N, K/4] (vpq_affine_qmv_w8g64_bf16)."""
    N, Kw = codes.shape
    K = Kw * 4
    M = x.numel() // K
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    with torch.cuda.device(x.device):
        check(lib().vpq_affine_qmv_w8g64_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x), _ptr(out),
                                              K, N, M, _stream(stream)))
    return out


def moe_gate_w8(codes, scales, biases, x, out=None, stream=None) -> torch.Tensor:
    """out[m] = sigmoid(dequant(w[1, K]) . x[m]) for one 8-bit row (vpq_affine_moe_gate_w8g64_bf16)."""
    K = codes.numel() * 4
    M = x.numel() // K
    if out is None:
        out = torch.empty((M,), dtype=torch.bfloat16, device=x.device)
    with torch.cuda.device(x.device):
        check(lib().vpq_affine_moe_gate_w8g64_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x), _ptr(out), K, M,
                                                   _stream(stream)))
    return out


def qmv_w8_fused(codes, scales, biases, x, y, store, stream=None, kind="w8"):
    """A GEMV with a fused store through one descriptor; `store` as in qmv_set, `y` the (first) output
    tensor. kind "w8": 8-bit weights (vpq_affine_qmv_w8g64_bf16_fused); "batch": w4 g64 rows sharing one
    weight stream (vpq_affine_qmv_batch_w4g64_bf16_fused); "g32": w4 g32 (vpq_affine_qmv_w4g32_bf16_fused);
    "q40": w4 g32 scale-only, `biases` may be None (vpq_affine_qmv_w4g32_q40_bf16_fused); "w8g32": 8-bit weights
    in groups of 32 (vpq_affine_qmv_w8g32_bf16_fused)."""
    N, Kw = codes.shape
    K = Kw * (4 if kind in ("w8", "w8g32") else 8)
    d = _lib.LinearDesc()
    d.w, d.scales, d.x, d.y = _ptr(codes), _ptr(scales), _ptr(x), _ptr(y)
    d.biases = _ptr(biases) if biases is not None else None
    d.K, d.N, d.M = K, N, x.numel() // K
    d.epilogue = EPILOGUES[store["epilogue"]]
    if store.get("aux") is not None:
        d.aux = _ptr(store["aux"])
    if store.get("y3") is not None:
        d.y3 = _ptr(store["y3"])
    d.q_rows, d.k_rows = store.get("q_rows", 0), store.get("k_rows", 0)
    fn = {"w8": lib().vpq_affine_qmv_w8g64_bf16_fused, "w8g32": lib().vpq_affine_qmv_w8g32_bf16_fused,
          "batch": lib().vpq_affine_qmv_batch_w4g64_bf16_fused,
          "g32": lib().vpq_affine_qmv_w4g32_bf16_fused, "q40": lib().vpq_affine_qmv_w4g32_q40_bf16_fused}[kind]
    with torch.cuda.device(x.device):
        check(fn(C.byref(d), _stream(stream)))
    return y


def qmv_batch_rows(codes, scales, biases, x, out=None, stream=None) -> torch.Tensor:
    """x [M, K] with small M: the rows share one stream of the weights (vpq_affine_qmv_batch_w4g64_bf16)."""
    N, Kw = codes.shape
    K = Kw * 8
    M = x.numel() // K
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    with torch.cuda.device(x.device):
        check(lib().vpq_affine_qmv_batch_w4g64_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x), _ptr(out),
                                                    K, N, M, _stream(stream)))
    return out


def qmv_add(codes, scales, biases, x, residual, out=None, stream=None) -> torch.Tensor:
    """y = bf16(bf16(x W^T) + residual) (vpq_affine_qmv_w4g64_bf16_add)."""
    N, Kw = codes.shape
    K = Kw * 8
    M = x.numel() // K
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    with torch.cuda.device(x.device):
        check(lib().vpq_affine_qmv_w4g64_bf16_add(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x), _ptr(out),
                                                  K, N, M, _ptr(residual), _stream(stream)))
    return out


def qmv_swiglu(codes, scales, biases, x, out=None, stream=None, act="swiglu") -> torch.Tensor:
    """Rows of W interleaved gate / up: y[M, N/2] = silu(gate) * up (vpq_affine_qmv_swiglu_w4g64_bf16),
    or gelu_tanh(gate) * up with act="geglu" (vpq_affine_qmv_geglu_w4g64_bf16)."""
    N, Kw = codes.shape
    K = Kw * 8
    M = x.numel() // K
    if out is None:
        out = torch.empty((M, N // 2), dtype=torch.bfloat16, device=x.device)
    fn = {"swiglu": lib().vpq_affine_qmv_swiglu_w4g64_bf16, "geglu": lib().vpq_affine_qmv_geglu_w4g64_bf16}[act]
    with torch.cuda.device(x.device):
        check(fn(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x), _ptr(out), K, N, M, _stream(stream)))
    return out


def qmv_geglu(codes, scales, biases, x, out=None, stream=None) -> torch.Tensor:
    return qmv_swiglu(codes, scales, biases, x, out, stream, act="geglu")


def qmv_gelu_mul(codes, scales, biases, x, mul, out=None, stream=None) -> torch.Tensor:
    """y = bf16(gelu_tanh(bf16(x W^T)) * mul) (vpq_affine_qmv_gelu_mul_w4g64_bf16)."""
    N, Kw = codes.shape
    K = Kw * 8
    M = x.numel() // K
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    with torch.cuda.device(x.device):
        check(lib().vpq_affine_qmv_gelu_mul_w4g64_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x),
                                                       _ptr(out), K, N, M, _ptr(mul), _stream(stream)))
    return out


def qmv_qkv(codes, scales, biases, x, q_rows, k_rows, v_rows, stream=None):
    """W = q | k | v row-concatenated; returns (q, k, v) (vpq_affine_qmv_qkv_w4g64_bf16)."""
    N, Kw = codes.shape
    K = Kw * 8
    M = x.numel() // K
    assert q_rows + k_rows + v_rows == N
    outs = [torch.empty((M, r), dtype=torch.bfloat16, device=x.device) for r in (q_rows, k_rows, v_rows)]
    with torch.cuda.device(x.device):
        check(lib().vpq_affine_qmv_qkv_w4g64_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x),
                                                  _ptr(outs[0]), _ptr(outs[1]) if k_rows else None,
                                                  _ptr(outs[2]) if v_rows else None, K, q_rows, k_rows, v_rows,
                                                  M, _stream(stream)))
    return tuple(outs)


EPILOGUES = {"none": 0, "add": 1, "swiglu": 2, "qkv": 3, "geglu": 4, "gelu_mul": 5, "silu_mul": 6}


def qmv_set(problems):
    """Builds the host descriptor array for qmv_batch / QmvPlan from (codes, scales, biases, x, y)
    tuples; an optional sixth element is a dict describing a fused store and the other options:
    {"epilogue": "add", "aux": residual} | {"epilogue": "swiglu"} | {"epilogue": "geglu"} |
    {"epilogue": "gelu_mul", "aux": mul} | {"epilogue": "silu_mul", "aux": mul} |
    {"epilogue": "qkv", "aux": k_out, "y3": v_out, "q_rows": .., "k_rows": ..};
    "norm_w": weights [K] and "eps" (RMSNorm of x while it is staged); "depends": True (plans: this
    GEMV reads what earlier entries write); "expert": int32 device tensor [M] with "x_div" (codes is
    then [E, N, K/8]: row m uses slab expert[m] and reads x row m // x_div); "M": rows, when x holds
    fewer rows than the descriptor has (expert gather)."""
    arr = (_lib.LinearDesc * len(problems))()
    for d, prob in zip(arr, problems):
        codes, scales, biases, x, y = prob[:5]
        e = prob[5] if len(prob) > 5 and prob[5] else {}
        N, Kw = codes.shape[-2], codes.shape[-1]
        d.w, d.scales, d.biases, d.x, d.y = _ptr(codes), _ptr(scales), _ptr(biases), _ptr(x), _ptr(y)
        d.K, d.N, d.M = Kw * 8, N, e.get("M", x.numel() // (Kw * 8))
        d.epilogue = EPILOGUES[e.get("epilogue", "none")]
        if e.get("aux") is not None:
            d.aux = _ptr(e["aux"])
        if e.get("y3") is not None:
            d.y3 = _ptr(e["y3"])
        d.q_rows, d.k_rows = e.get("q_rows", 0), e.get("k_rows", 0)
        d.depends = 1 if e.get("depends") else 0
        if e.get("norm_w") is not None:
            d.norm_w = _ptr(e["norm_w"])
            d.eps = float(e.get("eps", 1e-6))
        if e.get("expert") is not None:
            d.expert = _ptr(e["expert"])
            d.experts = codes.shape[0]
            d.x_div = int(e.get("x_div", 1))
            d.expert_div = int(e.get("expert_div", 1))
        if e.get("row_map") is not None:      # sorted slots: live iff row_map[m] >= 0; "row_gather": x row = row_map[m]
            d.row_map = _ptr(e["row_map"])
            d.row_gather = 1 if e.get("row_gather") else 0
    return arr


def qmv_batch(descs, stream=None) -> None:
    check(lib().vpq_affine_qmv_w4g64_bf16_batch(descs, len(descs), _stream(stream)))


def qmv_set_noalloc(descs, stream=None) -> None:
    """One launch for a set of at most 64 independent GEMV rows, with no device allocation and no
    workspace (vpq_affine_qmv_w4g64_bf16_set_noalloc). Calls must not overlap on the GPU."""
    check(lib().vpq_affine_qmv_w4g64_bf16_set_noalloc(descs, len(descs), _stream(stream)))


class QmvPlan:
    """A list of independent GEMVs run as one launch (vpq_qmv_plan_*). Holds the device workspace."""

    def __init__(self, problems, stream=None, workspace=None):
        self.descs = qmv_set(problems)
        self._keep = problems            # the plan captures pointers: keep the tensors alive
        dev = problems[0][0].device
        n = lib().vpq_qmv_plan_bytes(self.descs, len(self.descs))
        if workspace is not None and workspace.numel() < n:
            raise ValueError(f"QmvPlan: workspace of {workspace.numel()} bytes, {n} needed")
        self.workspace = workspace if workspace is not None else torch.empty(n, dtype=torch.uint8, device=dev)
        self.handle = C.c_void_p()
        with torch.cuda.device(dev):
            check(lib().vpq_qmv_plan_create(self.descs, len(self.descs), self.workspace.data_ptr(), self.workspace.numel(),
                                            _stream(stream), C.byref(self.handle)))

    def run(self, stream=None) -> None:
        check(lib().vpq_qmv_plan_run(self.handle, _stream(stream)))

    def close(self) -> None:
        if self.handle:
            lib().vpq_qmv_plan_destroy(self.handle)
            self.handle = None


def qmm(codes, scales, biases, x, out=None, stream=None) -> torch.Tensor:
    N, Kw = codes.shape
    K = Kw * 8
    M = x.numel() // K
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    with torch.cuda.device(x.device):
        check(lib().vpq_affine_qmm_w4g64_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x),
                                              _ptr(out), K, N, M, _stream(stream)))
    return out


def qmm_qkv(codes, scales, biases, x, q_rows, k_rows, v_rows, outs=None, stream=None):
    """W = q | k | v row-concatenated, one GEMM, three outputs (vpq_affine_qmm_qkv_w4g64_bf16)."""
    N, Kw = codes.shape
    K = Kw * 8
    M = x.numel() // K
    assert q_rows + k_rows + v_rows == N
    if outs is None:
        outs = [torch.empty((M, r), dtype=torch.bfloat16, device=x.device) for r in (q_rows, k_rows, v_rows)]
    with torch.cuda.device(x.device):
        check(lib().vpq_affine_qmm_qkv_w4g64_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x), _ptr(outs[0]),
                                                  _ptr(outs[1]), _ptr(outs[2]), K, q_rows, k_rows, v_rows, M,
                                                  _stream(stream)))
    return tuple(outs)


def qmm_any(codes, scales, biases, x, bits: int, group: int, act: str = "none", out=None, stream=None) -> torch.Tensor:
    """GEMM over any format twin (vpq_affine_qmm_bf16): bits 4 | 8, group 64 | 32, act "none" | "geglu"."""
    N, Kw = codes.shape
    K = Kw * (32 // bits)
    M = x.numel() // K
    a = {"none": 0, "geglu": 2}[act]
    if out is None:
        out = torch.empty((M, N // 2 if a else N), dtype=torch.bfloat16, device=x.device)
    with torch.cuda.device(x.device):
        check(lib().vpq_affine_qmm_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x), _ptr(out), K, N, M, bits,
                                        group, a, _stream(stream)))
    return out


def qmm_w8(codes, scales, biases, x, out=None, stream=None) -> torch.Tensor:
    """GEMM over 8-bit group-64 weights, codes int32 [N, K/4] (vpq_affine_qmm_w8g64_bf16)."""
    N, Kw = codes.shape
    K = Kw * 4
    M = x.numel() // K
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    with torch.cuda.device(x.device):
        check(lib().vpq_affine_qmm_w8g64_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x), _ptr(out),
                                              K, N, M, _stream(stream)))
    return out


def qmm_swiglu(codes, scales, biases, x, out=None, stream=None, act="swiglu", bits=4) -> torch.Tensor:
    """Rows of W interleaved gate / up: y[M, N/2] = act(gate) * up, act silu ("swiglu") or gelu_tanh
    ("geglu"), over 4- or 8-bit weights (vpq_affine_qmm_{swiglu,geglu}_w{4,8}g64_bf16)."""
    N, Kw = codes.shape
    K = Kw * (32 // bits)
    M = x.numel() // K
    if out is None:
        out = torch.empty((M, N // 2), dtype=torch.bfloat16, device=x.device)
    fn = getattr(lib(), f"vpq_affine_qmm_{act}_w{bits}g64_bf16")
    with torch.cuda.device(x.device):
        check(fn(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x), _ptr(out), K, N, M, _stream(stream)))
    return out


def qmm_swiglu_into(codes, scales, biases, x, out, out_off, bits=4, stream=None) -> torch.Tensor:
    """silu(gate) * up written into columns [out_off, out_off + N/2) of the row-major `out` [M, stride]
    (vpq_affine_qmm_swiglu_bf16_rs)."""
    N, Kw = codes.shape
    K = Kw * (32 // bits)
    M = x.numel() // K
    with torch.cuda.device(x.device):
        check(lib().vpq_affine_qmm_swiglu_bf16_rs(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x), _ptr(out), K, N,
                                                  M, bits, out.shape[-1], out_off, _stream(stream)))
    return out


def qmm_grouped_tile_rows() -> int:
    return int(lib().vpq_qmm_grouped_tile_rows())


def qmm_grouped_gated(codes, scales, biases, x, tile2e, srow=None, act="swiglu", out=None, stream=None, bits=4):
    """Gate|up GEMM of a mixture of experts over sorted, padded rows: codes [E, N, K*bits/32]; x the hidden
    [T, K] with srow [M] (gathered), or already sorted [M, K] with srow None. Returns y [M, N/2] in
    sorted order (vpq_affine_qmm_grouped_{swiglu,geglu}_w4g64_bf16; bits=8: vpq_affine_qmm_grouped_w8g64_bf16)."""
    E, N, Kw = codes.shape
    K = Kw * 32 // bits
    M = int(srow.numel()) if srow is not None else x.numel() // K
    if out is None:
        out = torch.empty((M, N // 2), dtype=torch.bfloat16, device=x.device)
    scratch = torch.empty((M, K), dtype=torch.bfloat16, device=x.device) if srow is not None else None
    args = (_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x), _ptr(out), K, N, M, _ptr(tile2e),
            _ptr(srow) if srow is not None else None, E, x.numel() // K,
            _ptr(scratch) if scratch is not None else None, _stream(stream))
    with torch.cuda.device(x.device):
        if bits == 8:
            check(lib().vpq_affine_qmm_grouped_w8g64_bf16({"swiglu": 1, "geglu": 2}[act], *args))
        else:
            check(getattr(lib(), f"vpq_affine_qmm_grouped_{act}_w4g64_bf16")(*args))
    return out


def qmm_grouped_down(codes, scales, biases, x_sorted, tile2e, sdst=None, y_rows=0, out=None, stream=None, bits=4):
    """Down GEMM of a mixture of experts: x_sorted [M, K]; row m of the product lands in row sdst[m]
    of y [y_rows, N] (vpq_affine_qmm_grouped_w4g64_bf16; bits=8: vpq_affine_qmm_grouped_w8g64_bf16). Rows of y
    no slot points at are not written."""
    E, N, Kw = codes.shape
    K = Kw * 32 // bits
    M = x_sorted.numel() // K
    rows = y_rows if sdst is not None else M
    if out is None:
        out = torch.zeros((rows, N), dtype=torch.bfloat16, device=x_sorted.device)
    with torch.cuda.device(x_sorted.device):
        if bits == 8:
            check(lib().vpq_affine_qmm_grouped_w8g64_bf16(0, _ptr(codes), _ptr(scales), _ptr(biases), _ptr(x_sorted),
                                                          _ptr(out), K, N, M, _ptr(tile2e),
                                                          _ptr(sdst) if sdst is not None else None, E, rows, None,
                                                          _stream(stream)))
        else:
            check(lib().vpq_affine_qmm_grouped_w4g64_bf16(_ptr(codes), _ptr(scales), _ptr(biases), _ptr(x_sorted),
                                                          _ptr(out), K, N, M, _ptr(tile2e),
                                                          _ptr(sdst) if sdst is not None else None, E, rows,
                                                          _stream(stream)))
    return out


# ---- the attention block between the q | k | v and the o projection
# A decode step makes these calls once a layer, so the checks below are written for a short way through Python.
_BF16, _I32, _I64, _F32 = torch.bfloat16, torch.int32, torch.int64, torch.float32
_DENSE = torch.contiguous_format
# torch's own short ways to the current stream and device; builds without CUDA do not bind them.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class _Placed:
    """Makes a device (and `stream`, if given) current for a call, so that what the call allocates belongs to the
    stream that it runs on."""
    __slots__ = ("ctx",)

    def __init__(self, dev, stream):
        self.ctx = torch.cuda.stream(stream) if stream is not None else torch.cuda.device(dev)

    def __enter__(self):
        self.ctx.__enter__()

    def __exit__(self, *exc):
        self.ctx.__exit__(*exc)


def _elsewhere(dev, stream) -> bool:
    """Whether a call for tensors of device `dev` has to switch to it or to `stream` first."""
    if dev < 0:
        raise ValueError("vpipe_b200.ops: rows must be bfloat16 on a CUDA device (no CPU path)")
    if stream is not None and stream.device.index != dev:
        raise ValueError(f"vpipe_b200.ops: the stream belongs to {stream.device}, the tensors to cuda:{dev}")
    return stream is not None or dev != _current_device()


def _heads(name, t, dev, shape):
    """Pointer and row stride (elements) of bfloat16 rows [M, heads, dim]: strides beyond the row's are the caller's."""
    if t.dtype is not _BF16 or t.get_device() != dev or t.shape != shape:
        raise ValueError(f"vpipe_b200.ops: {name} must be bfloat16 {tuple(shape)} on cuda:{dev} (no CPU path), "
                         f"not {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.is_contiguous():
        return t.data_ptr(), 0
    sm, sh, sd = t.stride()
    if sd != 1 or (sh != shape[2] and shape[1] > 1):
        raise ValueError(f"vpipe_b200.ops: the heads of a row of {name} must be contiguous")
    if shape[0] <= 1:
        return t.data_ptr(), 0
    if sm == 0:  # "dense" to the library
        raise ValueError(f"vpipe_b200.ops: the rows of {name} share their memory")
    return t.data_ptr(), sm


def _index(name, t, dev, dtype, shape):
    if t.dtype is not dtype or t.get_device() != dev or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"vpipe_b200.ops: {name} must be a contiguous {dtype} tensor {tuple(shape)} on cuda:{dev}")
    return t.data_ptr()


def _table(t, dev, B):
    """Pointer, row stride (entries; 0: one row) and columns of a page table. The library takes stride 0 as "dense", which
    rows that share their memory are not."""
    if t.dtype is not _I32 or t.get_device() != dev or t.dim() != 2 or t.shape[0] != B:
        raise ValueError(f"vpipe_b200.ops: page_table must be int32 [{B}, max_pages] on cuda:{dev}")
    pages = t.shape[1]
    sb, sp = t.stride()
    if (sp != 1 and pages > 1) or (B > 1 and sb < pages):
        raise ValueError("vpipe_b200.ops: the rows of page_table must be contiguous and must not overlap")
    return t.data_ptr(), sb if B > 1 else 0, pages


def _scale(scale):
    """The descriptor's scale, an f32 number: 0 says 1 / sqrt(head_dim), which what f32 has no number for must not become."""
    if scale is None:
        return 0.0
    if not 2.0 ** -126 <= scale <= 2.3586e38:
        raise ValueError("vpipe_b200.ops: scale must be from 2^-126 to 2.3586e38 (None: 1 / sqrt(head_dim))")
    return scale


class PagedKVCache:
    """The pages of a key-value cache: k, v [pages, kv_heads, page_size, head_dim], bfloat16, or uint8 codes with
    k_scales, v_scales bfloat16 [pages, kv_heads, page_size, head_dim / 64, 2] = (scale, bias). Any strides whose last
    is dense (k and v alike): [pages, page_size, kv_heads, head_dim] is `.transpose(1, 2)` away. Made once; the
    tensors are held, not copied (struct vpq_kv_cache)."""

    def __init__(self, k, v, k_scales=None, v_scales=None):
        quantised = k_scales is not None
        want = torch.uint8 if quantised else torch.bfloat16
        if (v_scales is not None) != quantised or k.dtype != want or v.dtype != want:
            raise ValueError("PagedKVCache: bfloat16 pages without scales, or uint8 codes with k_scales and v_scales")
        if any(t is not None and t.dim() >= 4 and t.stride(2) == 0 for t in (k, v, k_scales, v_scales)):
            raise ValueError("PagedKVCache: tokens share their memory")  # stride 0: "dense" to the library
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.device != v.device or not k.is_cuda:
            raise ValueError("PagedKVCache: k and v must be alike, [pages, kv_heads, page_size, head_dim] on a CUDA device")
        if k.numel() == 0:
            raise ValueError("PagedKVCache: at least one page")
        if k.stride(3) != 1:
            raise ValueError("PagedKVCache: the last dimension must be contiguous")
        pages, heads, size, dim = k.shape
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self.device, self.kv_heads, self.head_dim, self.page_size = k.device, heads, dim, size
        self.num_pages, self.bits = pages, 8 if quantised else 16
        d = self.desc = _lib.KvCache()
        d.k, d.v = k.data_ptr(), v.data_ptr()
        d.num_pages, d.page_size, d.kv_heads, d.head_dim, d.bits = pages, size, heads, dim, self.bits
        d.page_stride, d.head_stride, d.token_stride = k.stride()[:3]
        if quantised:
            shape = (pages, heads, size, dim // 64, 2)
            for s in (k_scales, v_scales):
                if s.dtype != torch.bfloat16 or tuple(s.shape) != shape or s.device != k.device or s.stride() != k_scales.stride():
                    raise ValueError(f"PagedKVCache: k_scales and v_scales must be bfloat16 {shape}, alike")
            if k_scales.stride(4) != 1 or (dim > 64 and k_scales.stride(3) != 2):
                raise ValueError("PagedKVCache: the scale pairs of a row must be contiguous")
            d.k_scales, d.v_scales = k_scales.data_ptr(), v_scales.data_ptr()
            d.scale_page_stride, d.scale_head_stride, d.scale_token_stride = k_scales.stride()[:3]
        self.ref = C.byref(d)
        self._dev = k.get_device()
        self._rows = k_scales if quantised else k  # a bfloat16 tensor of this device
        self._workspace = {}  # per number of query heads: a view of one element that has the workspace's size

    @classmethod
    def empty(cls, pages, page_size, kv_heads, head_dim, bits=16, device="cuda"):
        """Pages that hold nothing yet (the tokens of a sequence are defined by its length, not by the pages)."""
        shape = (pages, kv_heads, page_size, head_dim)
        if bits == 16:
            return cls(*(torch.empty(shape, dtype=torch.bfloat16, device=device) for _ in range(2)))
        if bits != 8:
            raise ValueError("PagedKVCache.empty: bits must be 16 or 8")
        codes = [torch.empty(shape, dtype=torch.uint8, device=device) for _ in range(2)]
        pairs = [torch.empty(shape[:3] + (head_dim // 64, 2), dtype=torch.bfloat16, device=device) for _ in range(2)]
        return cls(*codes, *pairs)


def _qk_desc(q, k, q_norm_w, k_norm_w, cos_sin, positions, eps, interleaved, dev, v, q_out, k_out):
    """Checked arguments as the bytes of a vpq_qk_desc, the number of rows, q_out and k_out (made here if None; with v
    there is no k_out)."""
    shape, kshape = q.shape, k.shape
    if len(shape) != 3 or len(kshape) != 3:
        raise ValueError("vpipe_b200.ops: q and k must be bfloat16 [rows, heads, head_dim]")
    M, hq, D = shape
    hkv = kshape[1]
    if kshape[0] != M or kshape[2] != D:
        kshape = (M, hkv, D)  # what _heads will say
    pq, sq = _heads("q", q, dev, shape)
    pk, sk = _heads("k", k, dev, kshape)
    pv = so = pj = sj = sv = wq = wk = pt = pp = rows = rot = 0
    if v is not None:
        pv, sv = _heads("v", v, dev, kshape)
    elif k_out is not None:
        pj, sj = _heads("k_out", k_out, dev, kshape)
    if q_out is not None:
        po, so = _heads("q_out", q_out, dev, shape)
    if q_norm_w is not None:
        wq = _index("q_norm_w", q_norm_w, dev, _BF16, (D,))
    if k_norm_w is not None:
        wk = _index("k_norm_w", k_norm_w, dev, _BF16, (D,))
    if cos_sin is not None:
        table = cos_sin.shape
        if len(table) != 2:
            raise ValueError("vpipe_b200.ops: cos_sin must be float32 [rows, rot_dim]")
        rows, rot = table
        pt = _index("cos_sin", cos_sin, dev, _F32, table)
    if positions is not None:
        pp = _index("positions", positions, dev, _I32, (M,))
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=_DENSE)
        po = q_out.data_ptr()
    if k_out is None and v is None:
        k_out = torch.empty_like(k, memory_format=_DENSE)
        pj = k_out.data_ptr()
    return _lib.QkDesc.pack(pq, pk, pv, po, pj, sq, sk, sv, so, sj, wq, wk, pt, pp, M, rows, hq, hkv, D, rot, interleaved,
                            eps), M, q_out, k_out


def qk_norm_rope(q, k, q_norm_w=None, k_norm_w=None, cos_sin=None, positions=None, eps=1e-6, interleaved=False,
                 q_out=None, k_out=None, stream=None):
    """Norm of queries and keys over each head, then the position rotation, in one pass (vpq_qk_norm_rope_bf16).
    q [M, q_heads, D], k [M, kv_heads, D] bfloat16, rows with any stride (parts of one q | k | v row are fine);
    cos_sin float32 [rows, rot_dim] = cos | sin of the pairs' angles; token m takes row positions[m] (int32; None: row
    m) and is left as it was if that is outside of the table. q_out / k_out may be q / k. Returns (q_out, k_out)."""
    dev = q.get_device()
    if _elsewhere(dev, stream):
        with _Placed(dev, stream):
            return qk_norm_rope(q, k, q_norm_w, k_norm_w, cos_sin, positions, eps, interleaved, q_out, k_out)
    d, M, q_out, k_out = _qk_desc(q, k, q_norm_w, k_norm_w, cos_sin, positions, eps, interleaved, dev, None, q_out, k_out)
    if M != 0:
        check(lib().vpq_qk_norm_rope_bf16(d, _raw_stream(dev)))
    return q_out, k_out


def qkv_norm_rope_store(q, k, v, q_norm_w, k_norm_w, cos_sin, positions, cache, slots, eps=1e-6, interleaved=False,
                        q_out=None, stream=None):
    """qk_norm_rope with the keys, and the values as they are, going straight into the cache: row m to slot slots[m]
    (int64; page * page_size + place; negative: nowhere) (vpq_qkv_norm_rope_store_bf16). Returns q_out."""
    dev = cache._dev
    if _elsewhere(dev, stream):
        with _Placed(dev, stream):
            return qkv_norm_rope_store(q, k, v, q_norm_w, k_norm_w, cos_sin, positions, cache, slots, eps, interleaved,
                                       q_out)
    d, M, q_out, _ = _qk_desc(q, k, q_norm_w, k_norm_w, cos_sin, positions, eps, interleaved, dev, v, q_out, None)
    s = _index("slots", slots, dev, _I64, (M,))
    if M != 0:
        check(lib().vpq_qkv_norm_rope_store_bf16(d, cache.ref, s, _raw_stream(dev)))
    return q_out


def kv_store(k, v, cache, slots, stream=None):
    """Rows k, v [M, kv_heads, head_dim] into slots [M] of the cache, quantised if it is (vpq_kv_store_bf16)."""
    dev = cache._dev
    if _elsewhere(dev, stream):
        with _Placed(dev, stream):
            return kv_store(k, v, cache, slots)
    shape = (k.shape[0], cache.kv_heads, cache.head_dim)
    pk, sk = _heads("k", k, dev, shape)
    pv, sv = _heads("v", v, dev, shape)
    s = _index("slots", slots, dev, _I64, shape[:1])
    if shape[0] != 0:
        check(lib().vpq_kv_store_bf16(cache.ref, pk, pv, sk, sv, s, shape[0], _raw_stream(dev)))


def kv_load(cache, slots, k_out=None, v_out=None, stream=None):
    """The values of slots [M]: (k, v) bfloat16 [M, kv_heads, head_dim], zeros for a slot outside of the cache
    (vpq_kv_load_bf16)."""
    dev = cache._dev
    if _elsewhere(dev, stream):
        with _Placed(dev, stream):
            return kv_load(cache, slots, k_out, v_out)
    M = slots.numel()
    s = _index("slots", slots, dev, _I64, (M,))
    shape = (M, cache.kv_heads, cache.head_dim)
    sk = sv = 0
    if k_out is None:
        k_out = cache._rows.new_empty(shape)
        pk = k_out.data_ptr()
    else:
        pk, sk = _heads("k_out", k_out, dev, shape)
    if v_out is None:
        v_out = torch.empty_like(k_out, memory_format=_DENSE)
        pv = v_out.data_ptr()
    else:
        pv, sv = _heads("v_out", v_out, dev, shape)
    if M != 0:
        check(lib().vpq_kv_load_bf16(cache.ref, pk, pv, sk, sv, s, M, _raw_stream(dev)))
    return k_out, v_out


def paged_attention(q, cache, page_table, seq_lens, scale=None, window=0, out=None, stream=None):
    """Attention of one new token per sequence over the cache (vpq_paged_attention_bf16): q [B, q_heads, head_dim],
    page_table int32 [B, max_pages] (rows with any stride: a slice of a wider table is fine), seq_lens int32 [B] (the new
    token's own key included), window 0 = all tokens.
    Lengths are read on the device, so a captured call serves any. The workspace is allocated per call on the stream
    that the call runs on."""
    dev = cache._dev
    if _elsewhere(dev, stream):
        with _Placed(dev, stream):
            return paged_attention(q, cache, page_table, seq_lens, scale, window, out)
    shape = q.shape
    if len(shape) != 3 or shape[2] != cache.head_dim:
        raise ValueError(f"vpipe_b200.ops: q must be bfloat16 [batch, q_heads, {cache.head_dim}]")
    B, hq, _ = shape
    pt, ts, pages = _table(page_table, dev, B)
    scale = 0.0 if scale is None else _scale(scale)
    if not 0 <= window < 1 << 31:
        raise ValueError("vpipe_b200.ops: window must be from 0 (all tokens) to 2^31 - 1")
    pq, sq = _heads("q", q, dev, shape)
    ps = _index("seq_lens", seq_lens, dev, _I32, (B,))
    so = 0
    if out is None:
        out = torch.empty_like(q, memory_format=_DENSE)
        po = out.data_ptr()
    else:
        po, so = _heads("out", out, dev, shape)
    if B == 0:
        return out
    L, d = lib(), _lib.PagedAttentionDesc.pack(pq, po, sq, so, pt, ps, ts, B, pages, hq, window, scale)
    like = cache._workspace.get(hq)  # its size goes by the heads alone
    if like is None:
        need = int(L.vpq_paged_attention_bytes(d, cache.ref))
        like = cache._rows.as_strided(((need + 1) // 2,), (0,))  # bfloat16: two bytes each
        if need:  # 0: this descriptor is refused below
            cache._workspace[hq] = like
    ws = torch.empty_like(like, memory_format=_DENSE)
    check(L.vpq_paged_attention_bf16(d, cache.ref, ws.data_ptr(), 2 * like.numel(), _raw_stream(dev)))
    return out


def device_status(stream=None) -> int:
    """Raises VpqError: TIMEOUT if a bounded device-side wait gave up, INDEX if the attention block met an index
    outside of its table; else 0."""
    detail = C.c_uint32(0)
    check(lib().vpq_device_status(_stream(stream), C.byref(detail)))
    return int(detail.value)


def function(library: str, entry: str):
    """The reference's load_library(name).function(entry); None if unknown."""
    return lib().vpq_function_lookup(library.encode(), entry.encode())


def dispatch(fn, buffers, K=0, N=0, M=0, clip=1.0, q_rows=0, k_rows=0, v_rows=0, out_stride=0, out_off=0,
             experts=0, rows=0, top_k=0, eps=0.0, stream=None) -> None:
    """One dispatch with the reference's slot numbering (see include/vpq.h). `buffers` is a list
    indexed by slot, or a dict {slot: tensor}."""
    a = _lib.DispatchArgs()
    items = buffers.items() if isinstance(buffers, dict) else enumerate(buffers)
    for i, t in items:
        a.buffers[i] = _ptr(t) if t is not None else None
    a.K, a.N, a.M, a.clip = K, N, M, clip
    a.q_rows, a.k_rows, a.v_rows = q_rows, k_rows, v_rows
    a.out_stride, a.out_off, a.experts, a.rows = out_stride, out_off, experts, rows
    a.top_k, a.eps = top_k, eps
    check(lib().vpq_dispatch(fn, C.byref(a), _stream(stream)))
