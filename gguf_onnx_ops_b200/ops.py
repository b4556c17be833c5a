"""Host-side mirror of the reference's ONNX Runtime custom-op interface for the hot path.

Each function takes the op's inputs (torch CUDA tensors, ``None`` for an omitted optional input
``""``) and attributes, validates them with the reference's constraints and messages, allocates
the outputs with the reference's shapes (as ``KernelContext::GetOutput`` would) and calls the
C ABI of libgguf_onnx_ops.so on the current torch CUDA stream.

    Q8Gemv(x, w, scales=None, gguf=1)                  -> y        src/bolt_ops.cu:1592-1643, :2018-2027
    Q4Gemv(x, w, scales=None, iq2=3)                   -> y        src/bolt_ops.cu:1592-1643, :2028-2037
    Nvfp4Gemv(x, w, w_scale, gscale, gguf=1)           -> y        src/bolt_ops.cu:1411-1469, :2004-2016
    Q8Embed(w, input_ids)                              -> out      src/bolt_ops.cu:1645-1690, :2038-2044
    RmsNorm(x, gamma, epsilon)                         -> y        src/bolt_ops.cu:1692-1864, :2045-2051
    SkipRmsNorm(x, skip, gamma, epsilon)               -> y, sum   src/bolt_ops.cu:1692-1864, :2052-2061
    Relu2(x)                                           -> y        src/bolt_ops.cu:700-726, :1997-2003
    MoeRouteGGUF(x, gate_w, bias, topk, scale)         -> idx, weights, scores    src/bolt_ops.cu:512-546
    MoeRoute(x, gate_w_bf16, bias, topk, scale)        -> idx, weights, scores    src/bolt_ops.cu:513-547, :1947
    MoeVerify(z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s=None, topk, iq2=3) -> out, h, part, meta
                                                                   src/bolt_ops.cu:1327-1409, :1981-1996
    MoeDecode(z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s, topk)            -> out, h, part
                                                                   src/bolt_ops.cu:664-699, :1967-1980
    MambaStep / MambaStepGGUF / MambaVerify / MambaVerifyGGUF       -> y, conv_state, ssm_state, xbc, ypre
                                                                   src/bolt_ops.cu:68-378, :1886-1946

The attention side of a decode / verify step has no counterpart in the reference (no attention op there) and follows the
same conventions:

    QkNormRope(qkv, q_gamma, k_gamma, cos, sin, positions, heads, kv_heads)    -> q, k
    KvCache(k, v, k_scale, v_scale)                                            the paged 8-bit cache
    KvCacheWrite(k, v, cache, page_table, lens, new_lens=None)                 in place
    KvCacheRead(cache, page_table, lens, rows)                                 -> k, v
    KvCacheAttention(q, cache, page_table, lens, new_lens=None, scale, window) -> out (, lse)
    DraftVerify(target_probs, draft_probs, draft_tokens, u_accept, u_sample)   -> accepted, tokens

Every weight layout of the GEMVs is implemented: the GGUF ones (``gguf=1`` / ``iq2=3``) and the
legacy split layouts (``gguf=0``, ``iq2`` in 0..2, through ``gguf_gemv_legacy``).  The lower-level
``*_into`` functions write into caller-provided outputs (no allocation), for graph capture and
benchmarking.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import check, load

Q8_0_BYTES, IQ2_XXS_BYTES, NVFP4_BYTES = 34, 66, 36


def _stream(stream=None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _raw_stream(t: torch.Tensor) -> int:
    """The current stream of t's device as the C ABI takes it (a stream object costs 3 us of host time a call)."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _current_device() -> int:
    """The device that launches go to, for tensors that are on one (torch.cuda.current_device, but for its initialisation)."""
    return torch._C._cuda_getDevice()


def _wrong_device(t, name: str, op: str) -> ValueError:
    return ValueError(f"{op}: tensors must be on one device" if t.is_cuda else f"{op}: {name} must be a CUDA tensor")


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _need(t, name, dtype, op):
    if t is None:
        raise ValueError(f"{op}: Missing required tensor input {name}")
    if not t.is_cuda:
        raise ValueError(f"{op}: {name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise ValueError(f"{op}: {name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{op}: {name} must be contiguous")


def _need_on(dev: int, t, name, dtype, op):
    """_need of a tensor on the device of the call's first one."""
    if t is None:
        raise ValueError(f"{op}: Missing required tensor input {name}")
    if t.get_device() != dev:
        raise _wrong_device(t, name, op)
    if t.dtype != dtype:
        raise ValueError(f"{op}: {name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{op}: {name} must be contiguous")


# ------------------------------------------------------------------------------------------------
# GEMVs
# ------------------------------------------------------------------------------------------------
def q8_0_gemv_into(x: torch.Tensor, w: torch.Tensor, y: torch.Tensor, R: int, N: int, K: int, stream=None) -> None:
    check(load().gguf_q8_0_gemv(_ptr(x), _ptr(w), _ptr(y), R, N, K, _stream(stream)))


def iq2_xxs_gemv_into(x: torch.Tensor, w: torch.Tensor, y: torch.Tensor, R: int, N: int, K: int, stream=None) -> None:
    check(load().gguf_iq2_xxs_gemv(_ptr(x), _ptr(w), _ptr(y), R, N, K, _stream(stream)))


def nvfp4_gemv_into(x, w, gscale, y, R: int, N: int, K: int, stream=None) -> None:
    check(load().gguf_nvfp4_gemv(_ptr(x), _ptr(w), _ptr(gscale), _ptr(y), R, N, K, _stream(stream)))


def _gemv_shapes(x: torch.Tensor, w: torch.Tensor):
    K = x.shape[-1]
    R = x.numel() // K if K else 0
    N = w.shape[0]
    return R, N, K


def gemv_legacy_into(layout: int, x, w, scales, gscale, y, R: int, N: int, K: int, stream=None) -> None:
    check(load().gguf_gemv_legacy(layout, _ptr(x), _ptr(w), _ptr(scales), _ptr(gscale), _ptr(y), R, N, K,
                                  _stream(stream)))


def _legacy(op, layout, x, w, scales, gscale=None):
    _need(x, "x", torch.bfloat16, op)
    _need(w, "w", torch.uint8, op)
    R, N, K = _gemv_shapes(x, w)
    y = torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=x.device)
    gemv_legacy_into(layout, x, w, scales, gscale, y, R, N, K)
    return y


def Q8Gemv(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor | None = None, gguf: int = 1) -> torch.Tensor:
    """y[..., N] = x[..., K] @ deq(W)^T.  gguf=1: raw GGUF Q8_0 blocks W [N, (K/32)*34]; gguf=0: the
    split layout W u8 [N, K/32, 32] = q + 128 with bf16 scales [N, K/32] (src/bolt_ops.cu:1617-1640)."""
    if gguf != 1:
        _need(w, "w", torch.uint8, "Q8Gemv")
        _need(scales, "scales", torch.bfloat16, "Q8Gemv")
        K = x.shape[-1]
        if K % 32 != 0 or w.dim() < 2 or w.shape[1] * 32 != K or w.numel() != w.shape[0] * K \
                or scales.numel() != w.shape[0] * (K // 32):
            raise ValueError("QGemv: K mismatch")
        return _legacy("Q8Gemv", _lib.GGUF_LAYOUT_Q8_SPLIT, x, w, scales)
    _need(x, "x", torch.bfloat16, "Q8Gemv")
    _need(w, "w", torch.uint8, "Q8Gemv")
    R, N, K = _gemv_shapes(x, w)
    if K % 64 != 0 or w.numel() != N * (K // 32) * Q8_0_BYTES or R < 1 or R > 16:
        raise ValueError("Q8Gemv gguf=1: needs B [N, (K/32)*34] and 1..16 rows")
    y = torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=x.device)
    q8_0_gemv_into(x, w, y, R, N, K)
    return y


def Q4Gemv(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor | None = None, iq2: int = 3) -> torch.Tensor:
    """y[..., N] = x[..., K] @ deq(W)^T.  iq2=3: raw GGUF IQ2_XXS super-blocks W [N, (K/256)*66];
    iq2=0: 4-bit W [N, K/32, 16] (n - 8) with bf16 scales [N, K/32]; iq2=1: 3-bit IQ2 codes in the
    same packing; iq2=2: IQ2_XXS records W [N, K/32, 8] with fp16 d bits [N, K/256] carried in a
    bf16-typed tensor (src/bolt_ops.cu:1593-1643)."""
    if iq2 != 3:
        if iq2 not in (0, 1, 2):
            raise NotImplementedError(f"Q4Gemv: unknown iq2={iq2}")
        _need(w, "w", torch.uint8, "Q4Gemv")
        _need(scales, "scales", torch.bfloat16, "Q4Gemv")
        K = x.shape[-1]
        N = w.shape[0]
        if iq2 == 2:
            if K % 256 != 0 or w.dim() != 3 or w.shape[1] * 32 != K or w.shape[2] != 8 or scales.numel() != N * (K // 256):
                raise ValueError("Q4Gemv iq2=2: needs B [N, K/32, 8] and 1..16 rows")
            layout = _lib.GGUF_LAYOUT_IQ2_NATIVE
        else:
            if K % 32 != 0 or w.dim() < 2 or w.shape[1] * 32 != K or w.numel() != N * K // 2 \
                    or scales.numel() != N * (K // 32):
                raise ValueError("QGemv: K mismatch")
            layout = _lib.GGUF_LAYOUT_IQ2_CODES if iq2 == 1 else _lib.GGUF_LAYOUT_Q4_SPLIT
        return _legacy("Q4Gemv", layout, x, w, scales)
    _need(x, "x", torch.bfloat16, "Q4Gemv")
    _need(w, "w", torch.uint8, "Q4Gemv")
    R, N, K = _gemv_shapes(x, w)
    if K % 256 != 0 or w.numel() != N * (K // 256) * IQ2_XXS_BYTES or R < 1 or R > 16:
        raise ValueError("Q4Gemv iq2=3: needs B [N, (K/256)*66] and 1..16 rows")
    y = torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=x.device)
    iq2_xxs_gemv_into(x, w, y, R, N, K)
    return y


def Nvfp4Gemv(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor | None, gscale: torch.Tensor,
              gguf: int = 1) -> torch.Tensor:
    """y[..., N] = gscale * (x[..., K] @ deq(W)^T).  gguf=1: raw GGUF NVFP4 blocks W [N, (K/64)*36];
    gguf=0: E2M1 nibbles W [N, K/2] with e4m3fn scales [N, K/16] (src/bolt_ops.cu:1411-1469)."""
    if gguf != 1:
        _need(w, "w", torch.uint8, "Nvfp4Gemv")
        _need(w_scale, "ws", torch.uint8, "Nvfp4Gemv")
        _need(gscale, "gscale", torch.float32, "Nvfp4Gemv")
        K = x.shape[-1]
        if K % 32 != 0 or w.dim() != 2 or w.shape[1] * 2 != K or w_scale.numel() != w.shape[0] * (K // 16):
            raise ValueError("Nvfp4Gemv: K mismatch (K % 32 required)")
        return _legacy("Nvfp4Gemv", _lib.GGUF_LAYOUT_NVFP4_SPLIT, x, w, w_scale, gscale)
    _need(x, "x", torch.bfloat16, "Nvfp4Gemv")
    _need(w, "w", torch.uint8, "Nvfp4Gemv")
    _need(gscale, "gscale", torch.float32, "Nvfp4Gemv")
    R, N, K = _gemv_shapes(x, w)
    if K % 64 != 0 or w.numel() != N * (K // 64) * NVFP4_BYTES or R < 1 or R > 16:
        raise ValueError("Nvfp4Gemv gguf=1: needs w [N, (K/64)*36] and 1..16 rows")
    y = torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=x.device)
    nvfp4_gemv_into(x, w, gscale, y, R, N, K)
    return y


# ------------------------------------------------------------------------------------------------
# Embedding
# ------------------------------------------------------------------------------------------------
def q8_0_embed_into(w, ids, out, vocab: int, row_bytes: int, R: int, stream=None) -> None:
    check(load().gguf_q8_0_embed(_ptr(w), _ptr(ids), _ptr(out), vocab, row_bytes, R, _stream(stream)))


def Q8Embed(w: torch.Tensor, input_ids: torch.Tensor) -> torch.Tensor:
    """Gather + dequantise rows of a raw GGUF Q8_0 table w [vocab, (K/32)*34] -> bf16 [..., K]
    (src/bolt_ops.cu:1645-1690, :2038-2044); out-of-range ids read row 0."""
    _need(w, "w", torch.uint8, "Q8Embed")
    _need(input_ids, "input_ids", torch.int64, "Q8Embed")
    vocab = w.shape[0]
    if vocab <= 0 or w.numel() % vocab != 0:
        raise ValueError("Q8Embed: invalid weight shape")
    row_bytes = w.numel() // vocab
    if row_bytes <= 0 or row_bytes % Q8_0_BYTES != 0:
        raise ValueError("Q8Embed: row_bytes must be a positive multiple of 34")
    K = row_bytes // Q8_0_BYTES * 32
    out = torch.empty(*input_ids.shape, K, dtype=torch.bfloat16, device=w.device)
    q8_0_embed_into(w, input_ids, out, vocab, row_bytes, input_ids.numel())
    return out


# ------------------------------------------------------------------------------------------------
# Norms
# ------------------------------------------------------------------------------------------------
def rms_norm_into(x, skip, gamma, y, sum_out, R: int, H: int, eps: float, stream=None) -> None:
    check(load().gguf_rms_norm(_ptr(x), _ptr(skip), _ptr(gamma), _ptr(y), _ptr(sum_out), R, H, eps, _stream(stream)))


def _norm_shapes(x, gamma, op):
    _need(x, "x", torch.bfloat16, op)
    _need(gamma, "gamma", torch.float32, op)
    if x.dim() < 1:
        raise ValueError(f"{op}: input must be at least 1D")
    H = x.shape[-1]
    if H <= 0 or H % 8 != 0:
        raise ValueError(f"{op}: hidden size H must be a positive multiple of 8")
    if gamma.numel() != H:
        raise ValueError(f"{op}: gamma size mismatch")
    return x.numel() // H, H


def RmsNorm(x: torch.Tensor, gamma: torch.Tensor, epsilon: float = 1e-5) -> torch.Tensor:
    """y = bf16(bf16(gamma) * x * rsqrt(mean(x^2) + eps)) over the last dim (src/bolt_ops.cu:1692-1864)."""
    R, H = _norm_shapes(x, gamma, "RmsNorm")
    y = torch.empty_like(x)
    rms_norm_into(x, None, gamma, y, None, R, H, epsilon)
    return y


def SkipRmsNorm(x: torch.Tensor, skip: torch.Tensor, gamma: torch.Tensor, epsilon: float = 1e-5,
                return_sum: bool = True):
    """sum = bf16(x + skip); y = RmsNorm(sum).  Returns (y, sum), or (y,) when the optional second
    output is not requested (src/bolt_ops.cu:1830-1856)."""
    R, H = _norm_shapes(x, gamma, "SkipRmsNorm")
    _need(skip, "skip", torch.bfloat16, "SkipRmsNorm")
    if skip.numel() != x.numel():
        raise ValueError("SkipRmsNorm: skip shape mismatch")
    y = torch.empty_like(x)
    s = torch.empty_like(x) if return_sum else None
    rms_norm_into(x, skip, gamma, y, s, R, H, epsilon)
    return (y, s) if return_sum else (y,)


def rms_norm_iq2_xxs_gemv_into(x, skip, gamma, eps, w, y, x_norm, sum_out, N: int, K: int, stream=None) -> None:
    check(load().gguf_rms_norm_iq2_xxs_gemv(_ptr(x), _ptr(skip), _ptr(gamma), eps, _ptr(w), _ptr(y), _ptr(x_norm),
                                            _ptr(sum_out), N, K, _stream(stream)))


def SkipRmsNormQ4Gemv(x: torch.Tensor, skip: torch.Tensor | None, gamma: torch.Tensor, w: torch.Tensor,
                      epsilon: float = 1e-5):
    """Fused decode step (an extension, not a reference op): y = Q4Gemv iq2=3(RmsNorm(x [+ skip])) for one
    row, K = 4096.  Returns (y [1, N], x_norm [1, K], sum [1, K] or None), bit-identical to SkipRmsNorm /
    RmsNorm followed by Q4Gemv."""
    _need(x, "x", torch.bfloat16, "SkipRmsNormQ4Gemv")
    _need(gamma, "gamma", torch.float32, "SkipRmsNormQ4Gemv")
    _need(w, "w", torch.uint8, "SkipRmsNormQ4Gemv")
    K = x.shape[-1]
    N = w.shape[0]
    if x.numel() != K or K != 4096 or gamma.numel() != K or w.numel() != N * (K // 256) * IQ2_XXS_BYTES:
        raise ValueError("SkipRmsNormQ4Gemv: needs one row of K = 4096 and w [N, (K/256)*66]")
    if skip is not None:
        _need(skip, "skip", torch.bfloat16, "SkipRmsNormQ4Gemv")
    y = torch.empty(1, N, dtype=torch.bfloat16, device=x.device)
    x_norm = torch.empty(1, K, dtype=torch.bfloat16, device=x.device)
    s = torch.empty(1, K, dtype=torch.bfloat16, device=x.device) if skip is not None else None
    rms_norm_iq2_xxs_gemv_into(x, skip, gamma, epsilon, w, y, x_norm, s, N, K)
    return y, x_norm, s


# ------------------------------------------------------------------------------------------------
# Router + MoE
# ------------------------------------------------------------------------------------------------
def moe_route_into(x, gate_w, bias, idx, weights, scores, R, K, E, topk, scale, stream=None) -> None:
    check(load().gguf_moe_route(_ptr(x), _ptr(gate_w), _ptr(bias), _ptr(idx), _ptr(weights), _ptr(scores),
                                R, K, E, topk, float(scale), _stream(stream)))


def MoeRouteGGUF(x: torch.Tensor, gate_w: torch.Tensor, bias: torch.Tensor, topk: int, scale: float):
    """Sigmoid router with F32 GGUF gate weights (rounded to bf16) and bias-corrected top-k."""
    _need(x, "x", torch.bfloat16, "MoeRouteGGUF")
    _need(gate_w, "gate_w", torch.float32, "MoeRouteGGUF")
    _need(bias, "bias", torch.float32, "MoeRouteGGUF")
    R, K = x.shape
    E = gate_w.shape[0]
    if E > 512 or K % 256 != 0 or topk > 32 or gate_w.shape[1] != K or bias.numel() != E:
        raise ValueError("MoeRoute: unsupported shape")
    idx = torch.empty(R, topk, dtype=torch.int32, device=x.device)
    wts = torch.empty(R, topk, dtype=torch.float32, device=x.device)
    scores = torch.empty(R, E, dtype=torch.float32, device=x.device)
    moe_route_into(x, gate_w, bias, idx, wts, scores, R, K, E, topk, scale)
    return idx, wts, scores


def moe_route_bf16_into(x, gate_w, bias, idx, wts, scores, R, K, E, topk, scale, stream=None) -> None:
    check(load().gguf_moe_route_bf16(_ptr(x), _ptr(gate_w), _ptr(bias), _ptr(idx), _ptr(wts), _ptr(scores), R, K, E,
                                     topk, scale, _stream(stream)))


def MoeRoute(x: torch.Tensor, gate_w: torch.Tensor, bias: torch.Tensor, topk: int, scale: float):
    """MoeRouteGGUF with bf16 gate weights (src/bolt_ops.cu:513-547, :1947-1956)."""
    _need(x, "x", torch.bfloat16, "MoeRoute")
    _need(gate_w, "gate_w", torch.bfloat16, "MoeRoute")
    _need(bias, "bias", torch.float32, "MoeRoute")
    R, K = x.shape
    E = gate_w.shape[0]
    if E > 512 or K % 256 != 0 or topk > 32 or gate_w.shape[1] != K or bias.numel() != E:
        raise ValueError("MoeRoute: unsupported shape")
    idx = torch.empty(R, topk, dtype=torch.int32, device=x.device)
    wts = torch.empty(R, topk, dtype=torch.float32, device=x.device)
    scores = torch.empty(R, E, dtype=torch.float32, device=x.device)
    moe_route_bf16_into(x, gate_w, bias, idx, wts, scores, R, K, E, topk, scale)
    return idx, wts, scores


def relu2_into(x, y, n: int, stream=None) -> None:
    check(load().gguf_relu2(_ptr(x), _ptr(y), n, _stream(stream)))


def Relu2(x: torch.Tensor) -> torch.Tensor:
    """y = bf16(max(x, 0)^2) elementwise (src/bolt_ops.cu:700-726)."""
    _need(x, "x", torch.bfloat16, "Relu2")
    y = torch.empty_like(x)
    relu2_into(x, y, x.numel())
    return y


def moe_verify_into(z, idx, w, fc1_w, fc2_w, out, h, part, meta, R, E, I, topk, stream=None) -> None:
    check(load().gguf_moe_verify_iq2_xxs(_ptr(z), _ptr(idx), _ptr(w), _ptr(fc1_w), _ptr(fc2_w), _ptr(out), _ptr(h),
                                         _ptr(part), _ptr(meta), R, E, I, topk, _stream(stream)))


def moe_legacy_into(layout, z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s, out, h, part, meta, R, E, I, topk,
                    stream=None) -> None:
    check(load().gguf_moe_legacy(layout, _ptr(z), _ptr(idx), _ptr(w), _ptr(fc1_w), _ptr(fc1_s), _ptr(fc2_w),
                                 _ptr(fc2_s), _ptr(out), _ptr(h), _ptr(part), _ptr(meta), R, E, I, topk,
                                 _stream(stream)))


_MOE_LAYOUTS = {0: _lib.GGUF_LAYOUT_Q4_SPLIT, 1: _lib.GGUF_LAYOUT_IQ2_CODES, 2: _lib.GGUF_LAYOUT_IQ2_NATIVE}


def _moe_legacy(op, z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s, topk, iq2, with_meta):
    for t, n, dt in ((z, "z", torch.bfloat16), (idx, "idx", torch.int32), (w, "weights", torch.float32),
                     (fc1_w, "fc1_w", torch.uint8), (fc1_s, "fc1_s", torch.bfloat16), (fc2_w, "fc2_w", torch.uint8),
                     (fc2_s, "fc2_s", torch.bfloat16)):
        _need(t, n, dt, op)
    R = z.shape[0]
    P = R * topk
    if with_meta and (R < 1 or R > 8 or P > 128):
        raise ValueError("MoeVerify: rows must be in [1,8] and rows*topk <= 128")
    if z.shape[1] != 1024:
        raise ValueError(f"{op}: latent size must be 1024")
    E, I = fc1_w.shape[0], fc1_w.shape[1]
    per32 = 8 if iq2 == 2 else 16
    gsz = 256 if iq2 == 2 else 32
    if I % gsz != 0 or fc1_w.numel() != E * I * 32 * per32 or fc2_w.numel() != E * 1024 * (I // 32) * per32 \
            or fc1_s.numel() != E * I * (1024 // gsz) or fc2_s.numel() != E * 1024 * (I // gsz):
        raise ValueError(f"{op}: bad inter size")
    out = torch.empty(R, 1024, dtype=torch.bfloat16, device=z.device)
    h = torch.empty(P, I, dtype=torch.bfloat16, device=z.device)
    part = torch.empty(P, 1024, dtype=torch.float32, device=z.device)
    meta = torch.empty(1 + P + P * 8, dtype=torch.int32, device=z.device) if with_meta else None
    moe_legacy_into(_MOE_LAYOUTS[iq2], z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s, out, h, part, meta, R, E, I, topk)
    return (out, h, part, meta) if with_meta else (out, h, part)


def MoeDecode(z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s, *, topk: int):
    """relu^2 MoE over 4-bit experts fc1_w [E, I, 512] / fc2_w [E, 1024, I/2] with bf16 scales per 32
    (src/bolt_ops.cu:664-699).  Returns (out [R,1024] bf16, h [R*topk, I] bf16, part [R*topk, 1024] f32)."""
    return _moe_legacy("MoeDecode", z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s, topk, 0, False)


def MoeVerify(z, idx, w, fc1_w, fc1_s=None, fc2_w=None, fc2_s=None, *, topk: int, iq2: int = 3):
    """Expert-grouped relu^2 MoE.  iq2=3: raw GGUF IQ2_XXS expert tensors; iq2=0: 4-bit experts with
    bf16 scales (as MoeDecode); iq2=1: 3-bit IQ2 codes; iq2=2: IQ2_XXS records + fp16 d
    (src/bolt_ops.cu:1327-1409).

    Returns (out [R,1024] bf16, h [R*topk, I] bf16, part [R*topk, 1024] f32, meta [1 + 9*R*topk] i32).
    """
    if iq2 in (0, 1, 2):
        return _moe_legacy("MoeVerify", z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s, topk, iq2, True)
    if iq2 != 3:
        raise NotImplementedError(f"MoeVerify: unknown iq2={iq2}")
    _need(z, "z", torch.bfloat16, "MoeVerify")
    _need(idx, "idx", torch.int32, "MoeVerify")
    _need(w, "weights", torch.float32, "MoeVerify")
    _need(fc1_w, "fc1_w", torch.uint8, "MoeVerify")
    _need(fc2_w, "fc2_w", torch.uint8, "MoeVerify")
    R = z.shape[0]
    P = R * topk
    if R < 1 or R > 8 or P > 128:
        raise ValueError("MoeVerify: rows must be in [1,8] and rows*topk <= 128")
    if z.shape[1] != 1024:
        raise ValueError("MoeVerify: latent size must be 1024")
    E, I = fc1_w.shape[0], fc1_w.shape[1]
    if I % 256 != 0 or fc1_w.numel() != E * I * (1024 // 256) * IQ2_XXS_BYTES \
            or fc2_w.numel() != E * 1024 * (I // 256) * IQ2_XXS_BYTES:
        raise ValueError("MoeVerify: inter size alignment mismatch")
    out = torch.empty(R, 1024, dtype=torch.bfloat16, device=z.device)
    h = torch.empty(P, I, dtype=torch.bfloat16, device=z.device)
    part = torch.empty(P, 1024, dtype=torch.float32, device=z.device)
    meta = torch.empty(1 + P + P * 8, dtype=torch.int32, device=z.device)
    moe_verify_into(z, idx, w, fc1_w, fc2_w, out, h, part, meta, R, E, I, topk)
    return out, h, part, meta


# ------------------------------------------------------------------------------------------------
# Mamba
# ------------------------------------------------------------------------------------------------
def mamba_step_into(proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, a_neg, d_skip, norm_w, state_row, y,
                    conv_out, ssm_out, xbc, ypre, *, R, state_rows, heads, n_groups, eps, tmin, stream=None) -> None:
    f32w = 1 if conv_w.dtype == torch.float32 else 0
    check(load().gguf_mamba_step(_ptr(proj), _ptr(conv_state), _ptr(ssm_state), _ptr(conv_w), _ptr(conv_b), f32w,
                                 _ptr(dt_bias), _ptr(a_neg), _ptr(d_skip), _ptr(norm_w), _ptr(state_row), _ptr(y),
                                 _ptr(conv_out), _ptr(ssm_out), _ptr(xbc), _ptr(ypre), R, state_rows, heads, 64, 128,
                                 n_groups, eps, tmin, _stream(stream)))


def _mamba(op, proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, a_neg, D, norm_w, state_row, *, heads, head_dim,
           d_state, n_groups, epsilon, time_step_min, gguf):
    wdt = torch.float32 if gguf else torch.bfloat16
    for t, n, dt in ((proj, "proj", torch.bfloat16), (conv_state, "conv_state", torch.bfloat16),
                     (ssm_state, "ssm_state", torch.float32), (conv_w, "conv_w", wdt), (conv_b, "conv_b", wdt),
                     (dt_bias, "dt_bias", torch.float32), (a_neg, "A_neg", torch.float32), (D, "D", torch.float32),
                     (norm_w, "norm_w", torch.float32)):
        _need(t, n, dt, op)
    if head_dim != 64 or d_state != 128:
        raise ValueError("MambaStep: only head_dim=64, d_state=128 are implemented")
    R = proj.shape[0]
    if R < 1 or R > 16:
        raise ValueError("MambaStep: rows must be in [1,16]")
    di = heads * head_dim
    cd = di + 2 * n_groups * d_state
    if proj.shape[1] != di + cd + heads:
        raise ValueError("MambaStep: bad proj width")
    if state_row is not None:
        _need(state_row, "state_row", torch.int32, op)
        if conv_state.shape[0] < R:
            raise ValueError("MambaVerify: state buffer needs >= R rows")
    dev = proj.device
    y = torch.empty(R, di, dtype=torch.bfloat16, device=dev)
    conv_out = torch.empty_like(conv_state)
    ssm_out = torch.empty_like(ssm_state)
    xbc = torch.empty(R, cd, dtype=torch.bfloat16, device=dev)
    ypre = torch.empty(R, di, dtype=torch.float32, device=dev)
    mamba_step_into(proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, a_neg, D, norm_w, state_row, y, conv_out,
                    ssm_out, xbc, ypre, R=R, state_rows=conv_state.shape[0], heads=heads, n_groups=n_groups,
                    eps=epsilon, tmin=time_step_min)
    return y, conv_out, ssm_out, xbc, ypre


def MambaStep(proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, A_neg, D, norm_w, *, heads, head_dim=64,
              d_state=128, n_groups, epsilon=1e-5, time_step_min=0.0):
    """One Mamba-2 mixer step (src/bolt_ops.cu:304-378).  Returns (y, conv_state_out, ssm_state_out,
    xbc_act, ypre)."""
    return _mamba("MambaStep", proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, A_neg, D, norm_w, None,
                  heads=heads, head_dim=head_dim, d_state=d_state, n_groups=n_groups, epsilon=epsilon,
                  time_step_min=time_step_min, gguf=False)


def MambaStepGGUF(proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, A_neg, D, norm_w, **attrs):
    """MambaStep with fp32 GGUF conv weights / bias (rounded to bf16 on use)."""
    return _mamba("MambaStepGGUF", proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, A_neg, D, norm_w, None,
                  gguf=True, **{"head_dim": 64, "d_state": 128, "epsilon": 1e-5, "time_step_min": 0.0, **attrs})


def MambaVerify(proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, A_neg, D, norm_w, state_row, **attrs):
    """MambaStep over R speculative tokens from state row *state_row; the state after token r is
    row r of the outputs (src/bolt_ops.cu:1915-1933)."""
    return _mamba("MambaVerify", proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, A_neg, D, norm_w, state_row,
                  gguf=False, **{"head_dim": 64, "d_state": 128, "epsilon": 1e-5, "time_step_min": 0.0, **attrs})


def MambaVerifyGGUF(proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, A_neg, D, norm_w, state_row, **attrs):
    """MambaVerify with fp32 GGUF conv weights / bias."""
    return _mamba("MambaVerifyGGUF", proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, A_neg, D, norm_w,
                  state_row, gguf=True,
                  **{"head_dim": 64, "d_state": 128, "epsilon": 1e-5, "time_step_min": 0.0, **attrs})


# ------------------------------------------------------------------------------------------------
# Attention: head norms and rotation, the 8-bit KV cache, draft verification
# ------------------------------------------------------------------------------------------------
def qk_norm_rope_into(x, q_gamma, k_gamma, cos, sin, positions, q, k, T: int, row_stride: int, heads: int, kv_heads: int,
                      head_dim: int, rot: int, max_pos: int, eps: float, interleaved: int, stream=None) -> None:
    rc = load().gguf_qk_norm_rope(x.data_ptr(), _ptr(q_gamma), _ptr(k_gamma), cos.data_ptr(), sin.data_ptr(),
                                  positions.data_ptr(), q.data_ptr(), k.data_ptr(), T, row_stride, heads, kv_heads, head_dim, rot,
                                  max_pos, eps, interleaved, _raw_stream(x) if stream is None else stream.cuda_stream)
    if rc:
        check(rc)


def QkNormRope(qkv: torch.Tensor, q_gamma: torch.Tensor | None, k_gamma: torch.Tensor | None, cos: torch.Tensor,
               sin: torch.Tensor, positions: torch.Tensor, *, heads: int, kv_heads: int, epsilon: float = 1e-6,
               interleaved: bool = False):
    """Per-head RMS norm of queries and keys (gamma f32 [head_dim], None: no norm) and rotation by the rows
    `positions` (int32 [T]) of cos / sin f32 [max_pos, rot / 2], in one pass and one rounding to bf16.

    qkv bf16 [..., (heads + 2 * kv_heads) * head_dim], T rows at one stride (queries, keys, values as one projection leaves
    them); the first rot values of a head turn as pairs (i, i + rot / 2), or (2i, 2i + 1) when interleaved.  Returns
    (q [..., heads, head_dim], k [..., kv_heads, head_dim]); a position outside the tables uses row 0 and is reported by
    device_status()."""
    dev = qkv.get_device()
    if dev < 0:
        raise ValueError("QkNormRope: qkv must be a CUDA tensor")
    if qkv.dtype != torch.bfloat16:
        raise ValueError(f"QkNormRope: qkv must be {torch.bfloat16}, got {qkv.dtype}")
    if qkv.dim() != 2 or qkv.stride(1) != 1:  # one row stride for all tokens, values side by side
        qkv2 = qkv.reshape(-1, qkv.shape[-1]) if qkv.is_contiguous() else None
        if qkv2 is None:
            raise ValueError("QkNormRope: qkv must be contiguous, or 2-D with contiguous rows")
    else:
        qkv2 = qkv
    T, width = qkv2.shape
    if heads < 1 or kv_heads < 1 or width % (heads + 2 * kv_heads) != 0:
        raise ValueError("QkNormRope: qkv width must be (heads + 2 * kv_heads) * head_dim")
    D = width // (heads + 2 * kv_heads)
    _need_on(dev, cos, "cos", torch.float32, "QkNormRope")
    _need_on(dev, sin, "sin", torch.float32, "QkNormRope")
    _need_on(dev, positions, "positions", torch.int32, "QkNormRope")
    if cos.dim() != 2 or cos.shape != sin.shape or positions.numel() != T:
        raise ValueError("QkNormRope: needs cos and sin [max_pos, rot / 2] and one position per row")
    for t, n in ((q_gamma, "q_gamma"), (k_gamma, "k_gamma")):
        if t is not None:
            _need_on(dev, t, n, torch.float32, "QkNormRope")
            if t.numel() != D:
                raise ValueError(f"QkNormRope: {n} size mismatch")
    if dev != _current_device():  # launches go there
        with torch.cuda.device(dev):
            return QkNormRope(qkv, q_gamma, k_gamma, cos, sin, positions, heads=heads, kv_heads=kv_heads, epsilon=epsilon,
                              interleaved=interleaved)
    lead = qkv.shape[:-1]
    q = qkv.new_empty((*lead, heads, D))
    k = qkv.new_empty((*lead, kv_heads, D))
    qk_norm_rope_into(qkv2, q_gamma, k_gamma, cos, sin, positions, q, k, T, qkv2.stride(0), heads, kv_heads, D,
                      2 * cos.shape[1], cos.shape[0], epsilon, 1 if interleaved else 0)
    return q, k


class KvCache:
    """The paged 8-bit cache of one attention layer: int8 codes k, v [pages, kv_heads, page, head_dim] and one f32 scale for
    each page and head, k_scale, v_scale [pages, kv_heads], not negative; a value is code * scale."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "pages", "kv_heads", "page", "head_dim", "device_index", "_c", "_ref")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        for t, n, dt in ((k, "k", torch.int8), (v, "v", torch.int8), (k_scale, "k_scale", torch.float32),
                         (v_scale, "v_scale", torch.float32)):
            _need(t, n, dt, "KvCache")
        if k.dim() != 4 or v.shape != k.shape or k_scale.shape != k.shape[:2] or v_scale.shape != k.shape[:2]:
            raise ValueError("KvCache: needs k, v [pages, kv_heads, page, head_dim] and scales [pages, kv_heads]")
        if len({t.device for t in (k, v, k_scale, v_scale)}) != 1:
            raise ValueError("KvCache: tensors must be on one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device_index = k.get_device()
        self.pages, self.kv_heads, self.page, self.head_dim = k.shape
        if self.page not in (16, 32, 64, 128, 256):
            raise ValueError("KvCache: page must be 16, 32, 64, 128 or 256 tokens")
        if self.head_dim not in (64, 96, 128, 192, 256):
            raise ValueError("KvCache: head_dim must be 64, 96, 128, 192 or 256")
        self._c = _lib.GgufKvCache(_ptr(k), _ptr(v), _ptr(k_scale), _ptr(v_scale), self.pages, self.kv_heads, self.page,
                                   self.head_dim)
        self._ref = ctypes.addressof(self._c)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page: int, head_dim: int, device) -> "KvCache":
        """A cache of zeros."""
        codes = [torch.zeros(pages, kv_heads, page, head_dim, dtype=torch.int8, device=device) for _ in range(2)]
        scales = [torch.zeros(pages, kv_heads, dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*codes, *scales)


def _kv_batch(op, cache, page_table, lens, new_lens):
    dev = cache.device_index
    _need_on(dev, page_table, "page_table", torch.int32, op)
    _need_on(dev, lens, "lens", torch.int32, op)
    B = lens.shape[0] if lens.dim() == 1 else -1
    if page_table.dim() != 2 or page_table.shape[0] != B:
        raise ValueError(f"{op}: needs page_table [B, pages of a sequence] and lens [B]")
    if new_lens is not None:
        _need_on(dev, new_lens, "new_lens", torch.int32, op)
        if new_lens.shape != lens.shape:
            raise ValueError(f"{op}: new_lens must have one number per sequence")
    return B, page_table.shape[1]


def _kv_rows(op, name, t, B, heads, cache):
    """The strides of t bf16 [B, R, heads, D] whose [heads, D] block is contiguous."""
    D = cache.head_dim
    if t.get_device() != cache.device_index:
        raise _wrong_device(t, name, op)
    if t.dtype != torch.bfloat16:
        raise ValueError(f"{op}: {name} must be {torch.bfloat16}, got {t.dtype}")
    if t.dim() != 4 or t.shape[0] != B or (heads and t.shape[2] != heads) or t.shape[3] != D:
        raise ValueError(f"{op}: {name} must be [B, rows, {heads or 'heads'}, {D}]")
    st = t.stride()
    if st[3] != 1 or (st[2] != D and t.shape[2] != 1):
        raise ValueError(f"{op}: the heads of a row of {name} must be contiguous")
    return st[0], st[1]


def kv_cache_write_into(cache: KvCache, k, v, page_table, lens, new_lens, B: int, R: int, cols: int, k_strides, v_strides,
                        stream=None) -> None:
    rc = load().gguf_kv_cache_write(cache._ref, k.data_ptr(), v.data_ptr(), page_table.data_ptr(), lens.data_ptr(), _ptr(new_lens),
                                    B, R, cols, *k_strides, *v_strides, _raw_stream(k) if stream is None else stream.cuda_stream)
    if rc:
        check(rc)


def KvCacheWrite(k: torch.Tensor, v: torch.Tensor, cache: KvCache, page_table: torch.Tensor, lens: torch.Tensor,
                 new_lens: torch.Tensor | None = None) -> None:
    """Quantises k, v bf16 [B, R, kv_heads, head_dim] (any strides of the first two dimensions) into the cache, in
    place, at positions lens[b] - n .. lens[b] - 1 of every sequence (n = new_lens[b], default R).

    For each touched page and head, with a = max |x| of the call's tokens there: s' = max(s, a / 127), s = 0 if the call
    begins the page; code = rint(x * (1 / s')); the page's older codes become rint(code * (s / s')).  A value that is not
    finite makes the scale NaN.  A shorter lens later (a rollback) needs no call; the scale stays."""
    B, cols = _kv_batch("KvCacheWrite", cache, page_table, lens, new_lens)
    ks = _kv_rows("KvCacheWrite", "k", k, B, cache.kv_heads, cache)
    vs = _kv_rows("KvCacheWrite", "v", v, B, cache.kv_heads, cache)
    if v.shape != k.shape:
        raise ValueError("KvCacheWrite: k and v must have the same shape")
    if cache.device_index != _current_device():
        with torch.cuda.device(cache.device_index):
            return KvCacheWrite(k, v, cache, page_table, lens, new_lens)
    kv_cache_write_into(cache, k, v, page_table, lens, new_lens, B, k.shape[1], cols, ks, vs)


def kv_cache_read_into(cache: KvCache, page_table, lens, k, v, B: int, rows: int, cols: int, stream=None) -> None:
    rc = load().gguf_kv_cache_read(cache._ref, page_table.data_ptr(), lens.data_ptr(), k.data_ptr(), v.data_ptr(), B, rows, cols,
                                   _raw_stream(k) if stream is None else stream.cuda_stream)
    if rc:
        check(rc)


def KvCacheRead(cache: KvCache, page_table: torch.Tensor, lens: torch.Tensor, *, rows: int):
    """The last `rows` tokens of every sequence as bf16: (k, v) [B, rows, kv_heads, head_dim]; row i is position
    lens[b] - rows + i, zeros where that is negative."""
    B, cols = _kv_batch("KvCacheRead", cache, page_table, lens, None)
    if rows < 0:
        raise ValueError("KvCacheRead: rows must be >= 0")
    if cache.device_index != _current_device():
        with torch.cuda.device(cache.device_index):
            return KvCacheRead(cache, page_table, lens, rows=rows)
    k = torch.empty(B, rows, cache.kv_heads, cache.head_dim, dtype=torch.bfloat16, device=cache.k.device)
    v = torch.empty_like(k)
    kv_cache_read_into(cache, page_table, lens, k, v, B, rows, cols)
    return k, v


class KvAttentionWorkspace:
    """Scratch of KvCacheAttention calls that do not overlap: partial results, and counters that are zero between calls.
    Grows to the largest call it has served.  What it has outgrown is kept as long as the workspace: a captured graph goes on
    using what it was captured with (so keep the workspace as long as the graph), and a call on another stream may not be
    done with it."""

    __slots__ = ("device", "scratch", "counters", "_sizes", "_captured", "_outgrown")

    def __init__(self, device, _captured: bool = False):
        self.device, self._captured = device, _captured
        self.scratch = self.counters = None
        self._sizes, self._outgrown = {}, []

    def fit(self, B: int, R: int, heads: int, kv_heads: int, head_dim: int) -> "KvAttentionWorkspace":
        key = (B, R, heads, kv_heads, head_dim)
        if key not in self._sizes:
            if not self._captured and torch.cuda.is_current_stream_capturing():  # its clearing would only be recorded
                raise ValueError("KvCacheAttention: call fit() of a workspace before it is used in a capture")
            nbytes, n = ctypes.c_int64(0), ctypes.c_int64(0)
            check(load().gguf_kv_cache_attention_workspace(*key, ctypes.byref(nbytes), ctypes.byref(n)))
            # (a handful of scratch sizes exist, and counters at least double: what is kept stays small)
            if self.scratch is None or self.scratch.numel() < nbytes.value:
                self._outgrown.append(self.scratch)
                self.scratch = torch.empty(nbytes.value, dtype=torch.uint8, device=self.device)
            if self.counters is None or self.counters.numel() < n.value:
                self._outgrown.append(self.counters)
                most = 1024 if self.counters is None else 2 * self.counters.numel()
                self.counters = torch.zeros(max(n.value, most), dtype=torch.int32, device=self.device)
            self._sizes[key] = True
        return self


_kv_workspaces: dict = {}


def _kv_workspace(device, stream) -> KvAttentionWorkspace:
    """The workspace kept for calls on this stream.  A call that is being captured gets one of its own, which the
    graph clears and uses at every replay."""
    if torch.cuda.is_current_stream_capturing():
        return KvAttentionWorkspace(device, _captured=True)
    key = (device, stream)
    ws = _kv_workspaces.get(key)
    if ws is None:
        ws = _kv_workspaces[key] = KvAttentionWorkspace(device)
    return ws


def kv_cache_attention_into(cache: KvCache, q, page_table, lens, new_lens, out, lse, workspace: KvAttentionWorkspace,
                            B: int, R: int, heads: int, cols: int, q_strides, scale: float, window: int,
                            stream=None) -> None:
    rc = load().gguf_kv_cache_attention(cache._ref, q.data_ptr(), page_table.data_ptr(), lens.data_ptr(), _ptr(new_lens),
                                        out.data_ptr(), _ptr(lse), workspace.scratch.data_ptr(), workspace.counters.data_ptr(), B, R,
                                        heads, cols, *q_strides, scale, window,
                                        _raw_stream(q) if stream is None else stream.cuda_stream)
    if rc:
        check(rc)


def KvCacheAttention(q: torch.Tensor, cache: KvCache, page_table: torch.Tensor, lens: torch.Tensor,
                     new_lens: torch.Tensor | None = None, *, scale: float | None = None, window: int = 0,
                     return_lse: bool = False, workspace: KvAttentionWorkspace | None = None):
    """Causal attention of the R newest tokens of every sequence over the cache: q bf16 [B, R, heads, head_dim] -> out of
    the same shape (and the log-sum-exp f32 [B, R, heads]).  Head h reads kv head h // (heads // kv_heads).

    lens[b] counts the new tokens; row r < n (n = new_lens[b], default R) sits at position lens[b] - n + r and sees itself and
    what is before it, or the last `window` positions of that.  Rows from n on give 0 (lse -inf).  scale defaults to
    head_dim ** -0.5.  One workspace is kept per device and stream; pass one to calls that share a stream with a
    captured graph's replay on another."""
    op = "KvCacheAttention"
    B, cols = _kv_batch(op, cache, page_table, lens, new_lens)
    strides = _kv_rows(op, "q", q, B, 0, cache)
    R, heads = q.shape[1], q.shape[2]
    if heads == 0 or heads % cache.kv_heads != 0:
        raise ValueError(f"{op}: heads must be a multiple of kv heads")
    if cache.device_index != _current_device():
        with torch.cuda.device(cache.device_index):
            return KvCacheAttention(q, cache, page_table, lens, new_lens, scale=scale, window=window, return_lse=return_lse,
                                    workspace=workspace)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty(B, R, heads, dtype=torch.float32, device=q.device) if return_lse else None
    ws = workspace if workspace is not None else _kv_workspace(q.device, _raw_stream(q))
    ws.fit(B, R, heads, cache.kv_heads, cache.head_dim)
    if ws.scratch.get_device() != cache.device_index:
        raise _wrong_device(ws.scratch, "workspace", op)
    kv_cache_attention_into(cache, q, page_table, lens, new_lens, out, lse, ws, B, R, heads, cols, strides,
                            cache.head_dim ** -0.5 if scale is None else scale, window)
    return (out, lse) if return_lse else out


def draft_verify_into(target, draft_probs, draft, u_accept, u_sample, drafts, accepted, tokens, B: int, R: int, V: int,
                      stream=None) -> None:
    rc = load().gguf_draft_verify(target.data_ptr(), _ptr(draft_probs), draft.data_ptr(), u_accept.data_ptr(), u_sample.data_ptr(),
                                  _ptr(drafts), accepted.data_ptr(), tokens.data_ptr(), B, R, V,
                                  _raw_stream(target) if stream is None else stream.cuda_stream)
    if rc:
        check(rc)


def DraftVerify(target_probs: torch.Tensor, draft_probs: torch.Tensor | None, draft_tokens: torch.Tensor,
                u_accept: torch.Tensor, u_sample: torch.Tensor, drafts: torch.Tensor | None = None):
    """Which drafted tokens stand against the target's probabilities, and the token after them.

    target_probs f32 [B, R + 1, V]; draft_probs f32 [B, R, V], or None for a drafter that was certain; draft_tokens int32
    [B, R]; u_accept f32 [B, R] and u_sample f32 [B] in [0, 1); drafts int32 [B]: drafts of each sequence (default R).
    Draft i stands iff u_accept * draft_probs(x_i) < target_probs(x_i); the next token is drawn from
    max(target - draft, 0) after a rejected draft, else from the target's row (include/gguf_ops.h says how, in whole
    numbers).  Returns (accepted int32 [B], tokens int32 [B, R + 1]: the drafts that stand, the next token, -1 after it);
    accepted[b] is the state_row of the sequence's next MambaVerify."""
    op = "DraftVerify"
    _need(target_probs, "target_probs", torch.float32, op)
    dev = target_probs.get_device()
    _need_on(dev, draft_tokens, "draft_tokens", torch.int32, op)
    _need_on(dev, u_accept, "u_accept", torch.float32, op)
    _need_on(dev, u_sample, "u_sample", torch.float32, op)
    if draft_tokens.dim() != 2 or target_probs.dim() != 3:
        raise ValueError(f"{op}: needs target_probs [B, R + 1, V] and draft_tokens [B, R]")
    B, R = draft_tokens.shape
    V = target_probs.shape[2]
    if target_probs.shape[:2] != (B, R + 1) or u_accept.shape != draft_tokens.shape or u_sample.shape != (B,):
        raise ValueError(f"{op}: needs target_probs [B, R + 1, V], u_accept [B, R] and u_sample [B]")
    if draft_probs is not None:
        _need_on(dev, draft_probs, "draft_probs", torch.float32, op)
        if draft_probs.shape != (B, R, V):
            raise ValueError(f"{op}: draft_probs must be [B, R, V]")
    if drafts is not None:
        _need_on(dev, drafts, "drafts", torch.int32, op)
        if drafts.shape != (B,):
            raise ValueError(f"{op}: drafts must have one number per sequence")
    if dev != _current_device():
        with torch.cuda.device(dev):
            return DraftVerify(target_probs, draft_probs, draft_tokens, u_accept, u_sample, drafts)
    accepted = draft_tokens.new_empty((B,))
    tokens = draft_tokens.new_empty((B, R + 1))
    draft_verify_into(target_probs, draft_probs, draft_tokens, u_accept, u_sample, drafts, accepted, tokens, B, R, V)
    return accepted, tokens


# ------------------------------------------------------------------------------------------------
# Debug / parity
# ------------------------------------------------------------------------------------------------
def dequantize(w: torch.Tensor, gguf_type: int, K: int) -> torch.Tensor:
    """Raw GGUF rows [rows, row_bytes] -> f32 [rows, K] with the GEMV's device decoders."""
    rows = w.shape[0]
    out = torch.empty(rows, K, dtype=torch.float32, device=w.device)
    check(load().gguf_dequantize(gguf_type, _ptr(w), _ptr(out), rows, K, _stream()))
    return out


def set_pdl(enable: bool) -> None:
    load().gguf_set_pdl(1 if enable else 0)


def set_fast_paths(enable) -> None:
    """Enable / disable the shape-specialised kernels (the generic engine handles every shape).

    ``True`` / 1 = on (default), ``False`` / 0 = generic engine only, 2 = on, with the bf16 instead of
    the integer tensor-core kernel for single-row IQ2_XXS (a cross-check of the two decoders)."""
    load().gguf_set_fast_paths(int(enable) if not isinstance(enable, bool) else (1 if enable else 0))


def device_status():
    return _lib.device_status()
