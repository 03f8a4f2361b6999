"""Tensor-level front end of the C ABI: thin argument checking, no arithmetic of its own."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import (CODE_HASH, CODE_LITE, CODE_LUT, LAYOUT_CHUNKED, LAYOUT_ROWMAJOR, LAYOUT_TILED, LAYOUT_UNITMAJOR,
                  XORDER_NATURAL, Format, call, check, lib, ptr, native)


def _cuda_contig(t: torch.Tensor, name: str, dtype: torch.dtype | None = None) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"{name} must have dtype {dtype}, got {t.dtype}")


def _ld(t: torch.Tensor, width: int) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(width, t.stride(0))


def units_per_row(n: int, K: int) -> int:
    if (n * K) % 128:
        raise RuntimeError(f"n*K = {n * K} bits per row is not a whole number of 128-bit units")
    return n * K // 128


def codes_shape(m: int, n: int, K: int, layout: int) -> tuple[int, ...]:
    nu = units_per_row(n, K)
    if layout == LAYOUT_ROWMAJOR:
        return (m, nu * 4)
    if layout == LAYOUT_CHUNKED:
        return (nu // 32, m, 128)
    if layout == LAYOUT_UNITMAJOR:
        return (nu, m, 4)
    return (m // 32, nu, 32, 4)


def repack(codes: torch.Tensor, src_layout: int, dst_layout: int, m: int, n_units: int) -> torch.Tensor:
    """Packed codes in `src_layout` -> a new tensor in `dst_layout` (rptc_repack)."""
    _cuda_contig(codes, "codes", torch.int32)
    if codes.numel() != m * n_units * 4:
        raise RuntimeError("codes has the wrong number of elements")
    if dst_layout == LAYOUT_ROWMAJOR:
        shape = (m, n_units * 4)
    elif dst_layout == LAYOUT_CHUNKED:
        shape = (n_units // 32, m, 128)
    elif dst_layout == LAYOUT_UNITMAJOR:
        shape = (n_units, m, 4)
    else:
        shape = (m // 32, n_units, 32, 4)
    out = torch.empty(shape, dtype=torch.int32, device=codes.device)
    call("rptc_repack", codes.device, ptr(codes), src_layout, ptr(out), dst_layout, m, n_units)
    return out


def decompress(codes: torch.Tensor, lut: torch.Tensor, m: int, n: int, fmt: Format, out: torch.Tensor | None = None,
               carry_in: torch.Tensor | None = None) -> torch.Tensor:
    """Packed codes -> dense fp16 [m, n] (rptc_decompress)."""
    if out is not None and carry_in is None:
        status = native().decompress(codes, lut, m, n, fmt, out)      # None: something is not as the kernel reads it
        if status is not None:
            check(status, "rptc_decompress")
            return out
    _cuda_contig(codes, "codes", torch.int32)
    _cuda_contig(lut, "lut", torch.float16)
    if lut.numel() != fmt.lut_numel():
        raise RuntimeError(f"lut must have {fmt.lut_numel()} elements, got {lut.numel()}")
    if codes.numel() * 32 != m * n * fmt.K:
        raise RuntimeError("codes has the wrong number of elements for m, n, K")
    if out is None:
        out = torch.empty((m, n), dtype=torch.float16, device=codes.device)
    else:
        if not out.is_cuda or out.dtype != torch.float16 or out.dim() != 2 or out.shape != (m, n) or out.stride(1) != 1:
            raise RuntimeError("out must be a CUDA fp16 [m, n] tensor with unit column stride")
    if carry_in is not None:
        _cuda_contig(carry_in, "carry_in", torch.int32)
    call("rptc_decompress", codes.device, ptr(codes), ptr(lut), ptr(carry_in), ptr(out), out.stride(0), m, n, ctypes.byref(fmt))
    return out


def check_alphabet(alphabet: torch.Tensor) -> None:
    if alphabet.dim() != 1 or alphabet.shape[0] not in [1 << L for L in range(3, 17)]:
        raise RuntimeError(f"the alphabet must be one row of 2^L entries, L = 3 to 16, got {tuple(alphabet.shape)}")


def dequantize(alphabet: torch.Tensor, symbols: torch.Tensor) -> torch.Tensor:
    """2-bit symbols int32 [rows, length] -> alphabet[state], rounded to fp16, in the alphabet's dtype (fp16 or fp32)
    (rptc_dequantize)."""
    _cuda_contig(alphabet, "alphabet")
    _cuda_contig(symbols, "symbols", torch.int32)
    if alphabet.dtype not in (torch.float16, torch.float32):
        raise RuntimeError("alphabet must be fp16 or fp32")
    check_alphabet(alphabet)
    rows, length = symbols.shape
    out = torch.empty((rows, length), dtype=alphabet.dtype, device=symbols.device)
    if out.numel():
        call("rptc_dequantize", symbols.device, alphabet.data_ptr(), symbols.data_ptr(), out.data_ptr(), int(alphabet.dtype == torch.float32), rows,
             length, alphabet.numel().bit_length() - 1)
    return out


def pack_symbols(symbols: torch.Tensor, bits: int, row_words: int) -> torch.Tensor:
    """Symbols int32 [rows, length] -> ROWMAJOR words int32 [rows, row_words], first symbol on top (rptc_pack_symbols)."""
    _cuda_contig(symbols, "symbols", torch.int32)
    rows, length = symbols.shape
    words = torch.empty((rows, row_words), dtype=torch.int32, device=symbols.device)
    call("rptc_pack_symbols", symbols.device, ptr(symbols), ptr(words), rows, length, row_words, bits)
    return words


def gemv_acc(codes: torch.Tensor, lut: torch.Tensor, x: torch.Tensor, acc: torch.Tensor, m: int, n: int, fmt: Format,
             x_order: int = XORDER_NATURAL, carry_in: torch.Tensor | None = None) -> None:
    """acc[b, :m] += W x[b]  (fp32 accumulator; rptc_gemv).  x: fp16 [b, n] or [n]."""
    _cuda_contig(codes, "codes", torch.int32)
    _cuda_contig(lut, "lut", torch.float16)
    if x.dim() == 1:
        x = x.unsqueeze(0)
    if acc.dim() == 1:
        acc = acc.unsqueeze(0)
    if not x.is_cuda or x.dtype != torch.float16 or x.stride(1) != 1 or x.shape[1] != n:
        raise RuntimeError("x must be a CUDA fp16 [batch, n] tensor with unit column stride")
    if not acc.is_cuda or acc.dtype != torch.float32 or acc.stride(1) != 1 or acc.shape[1] < m or acc.shape[0] != x.shape[0]:
        raise RuntimeError("acc must be a CUDA fp32 [batch, >=m] tensor")
    if codes.numel() * 32 != m * n * fmt.K:
        raise RuntimeError("codes has the wrong number of elements for m, n, K")
    if lut.numel() != fmt.lut_numel():
        raise RuntimeError(f"lut must have {fmt.lut_numel()} elements, got {lut.numel()}")
    call("rptc_gemv", codes.device, ptr(codes), ptr(lut), ptr(carry_in), ptr(x), x.stride(0) if x.shape[0] > 1 else max(n, x.stride(0)),
         ptr(acc), acc.stride(0) if acc.shape[0] > 1 else max(m, acc.stride(0)), m, n, x.shape[0], x_order, ctypes.byref(fmt))


def gemv_norm_input(codes: torch.Tensor, lut: torch.Tensor, acc: torch.Tensor, m: int, n: int, fmt: Format, rows: int,
                    prev_acc: torch.Tensor | None, signs_out: torch.Tensor | None, scale_out: float, h_in: torch.Tensor,
                    h_out: torch.Tensor, w_norm: torch.Tensor, eps: float, signs_in: torch.Tensor | None,
                    clear: torch.Tensor | None = None, carry_in: torch.Tensor | None = None) -> None:
    """acc += W x with x = H(s_in * rmsnorm(h_in + s_out * H(prev_acc) * scale_out) * w_norm), computed inside the
    launch; the updated residual goes to h_out (rptc_gemv_glued).  `clear` is zeroed by the launch."""
    from ._lib import GemvInput
    d = GemvInput(ptr(prev_acc), 0 if prev_acc is None else _ld(prev_acc, n), ptr(signs_out), scale_out, eps,
                  ptr(signs_in), ptr(h_in), ptr(h_out), _ld(h_in, n), ptr(w_norm), ptr(clear), 0 if clear is None else clear.numel())
    call("rptc_gemv_glued", codes.device, ptr(codes), ptr(lut), ptr(carry_in), ctypes.byref(d), ptr(acc), _ld(acc, m), m, n, rows,
         ctypes.byref(fmt))


def gemv_swiglu_input(codes: torch.Tensor, lut: torch.Tensor, acc: torch.Tensor, m: int, n: int, fmt: Format, rows: int,
                      prev_acc: torch.Tensor, signs_out: torch.Tensor | None, scale_out: float, signs_in: torch.Tensor | None,
                      block: int, clear: torch.Tensor | None = None, carry_in: torch.Tensor | None = None) -> None:
    """acc += W x with x = H(s_in * silu(g) * u), (g | u) = s_out * H(prev_acc) * scale_out, made inside the launch
    block by block (rptc_gemv_swiglu).  `clear` is zeroed by the launch."""
    call("rptc_gemv_swiglu", codes.device, ptr(codes), ptr(lut), ptr(carry_in), ptr(prev_acc), _ld(prev_acc, 2 * n), ptr(signs_out),
         scale_out, ptr(signs_in), block, ptr(acc), _ld(acc, m), m, n, rows, ctypes.byref(fmt), ptr(clear),
         0 if clear is None else clear.numel())


def gemv_finish(acc: torch.Tensor, y: torch.Tensor, m: int, scale: float = 1.0, accumulate: bool = False,
                clear: bool = True) -> None:
    """y = fp16(scale * acc) (+ y); optionally zero acc (rptc_gemv_finish)."""
    if acc.dim() == 1:
        acc = acc.unsqueeze(0)
    if y.dim() == 1:
        y = y.unsqueeze(0)
    call("rptc_gemv_finish", acc.device, ptr(acc), acc.stride(0) if acc.shape[0] > 1 else max(m, acc.stride(0)), ptr(y),
         y.stride(0) if y.shape[0] > 1 else max(m, y.stride(0)), m, acc.shape[0], scale, int(accumulate), int(clear))


def gemv(codes: torch.Tensor, lut: torch.Tensor, x: torch.Tensor, m: int, n: int, fmt: Format,
         x_order: int = XORDER_NATURAL, carry_in: torch.Tensor | None = None) -> torch.Tensor:
    """Convenience: allocate a zeroed fp32 accumulator, run the fused matvec, return fp16 [b, m]."""
    xb = x.unsqueeze(0) if x.dim() == 1 else x
    acc = torch.zeros((xb.shape[0], m), dtype=torch.float32, device=x.device)
    gemv_acc(codes, lut, xb, acc, m, n, fmt, x_order, carry_in)
    y = torch.empty((xb.shape[0], m), dtype=torch.float16, device=x.device)
    gemv_finish(acc, y, m, clear=False)
    return y[0] if x.dim() == 1 else y


def gemm(codes: torch.Tensor, lut: torch.Tensor, x: torch.Tensor, m: int, n: int, fmt: Format,
         out: torch.Tensor | None = None, carry_in: torch.Tensor | None = None, invariant: bool = False) -> torch.Tensor:
    """y[t] = W x[t] for a block of tokens on the tensor cores (rptc_gemm).  x: fp16 [tokens, n].  `invariant`: a token's
    result does not depend on the number of tokens (rptc_gemm_invariant)."""
    _cuda_contig(codes, "codes", torch.int32)
    _cuda_contig(lut, "lut", torch.float16)
    if not x.is_cuda or x.dtype != torch.float16 or x.dim() != 2 or x.stride(1) != 1 or x.shape[1] != n:
        raise RuntimeError("x must be a CUDA fp16 [tokens, n] tensor with unit column stride")
    if out is None:
        out = torch.empty((x.shape[0], m), dtype=torch.float16, device=x.device)
    call("rptc_gemm_invariant" if invariant else "rptc_gemm", codes.device, ptr(codes), ptr(lut), ptr(carry_in), ptr(x), x.stride(0), ptr(out),
         out.stride(0), m, n, x.shape[0], ctypes.byref(fmt))
    return out


def hadamard(x: torch.Tensor, signs: torch.Tensor | None, block: int, transpose: bool = False, scale: float = 1.0,
             out: torch.Tensor | None = None, clear_in: bool = False, residual: torch.Tensor | None = None) -> torch.Tensor:
    """Block-diagonal randomized Hadamard transform along the last axis (rptc_hadamard).

    x: fp16 or fp32 [rows, n]; result fp16 [rows, n] (+ residual)."""
    squeeze = x.dim() == 1
    if squeeze:
        x = x.unsqueeze(0)
    if not x.is_cuda or x.dim() != 2 or x.stride(1) != 1 or x.dtype not in (torch.float16, torch.float32):
        raise RuntimeError("x must be a CUDA fp16/fp32 [rows, n] tensor with unit column stride")
    rows, n = x.shape
    if out is None:
        out = torch.empty((rows, n), dtype=torch.float16, device=x.device)
    if signs is not None:
        _cuda_contig(signs, "signs", torch.float16)
    if residual is not None and residual.dim() == 1:
        residual = residual.unsqueeze(0)
    call("rptc_hadamard", x.device, ptr(x), int(x.dtype == torch.float32), _ld(x, n), ptr(out), _ld(out, n), ptr(signs), ptr(residual),
         0 if residual is None else _ld(residual, n), rows, n, block, int(transpose), scale, int(clear_in))
    return out[0] if squeeze else out


def swiglu_hadamard(acc: torch.Tensor, out: torch.Tensor, signs_out: torch.Tensor | None, signs_in: torch.Tensor | None,
                    n: int, block: int, scale_out: float, scale_in: float = 1.0, clear: bool = True) -> torch.Tensor:
    """Fused gated-MLP middle (rptc_swiglu_hadamard): acc fp32 [rows, 2n] -> out fp16 [rows, n]."""
    call("rptc_swiglu_hadamard", acc.device, ptr(acc), _ld(acc, 2 * n), ptr(out), _ld(out, n), ptr(signs_out), ptr(signs_in),
         acc.shape[0], n, block, scale_out, scale_in, int(clear))
    return out


def swiglu_hadamard_f16(gate_up: torch.Tensor, out: torch.Tensor, signs_out: torch.Tensor | None, signs_in: torch.Tensor | None,
                        n: int, block: int, scale_out: float, scale_in: float = 1.0) -> torch.Tensor:
    """Fused gated-MLP middle from the fp16 output of a matrix product (rptc_swiglu_hadamard_f16):
    gate_up fp16 [rows, 2n] -> out fp16 [rows, n]."""
    call("rptc_swiglu_hadamard_f16", gate_up.device, ptr(gate_up), _ld(gate_up, 2 * n), ptr(out), _ld(out, n), ptr(signs_out),
         ptr(signs_in), gate_up.shape[0], n, block, scale_out, scale_in)
    return out


def rmsnorm(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor, eps: float) -> torch.Tensor:
    rows, n = x.shape
    call("rptc_rmsnorm", x.device, ptr(x), _ld(x, n), ptr(w), ptr(out), _ld(out, n), rows, n, eps)
    return out


def rope_cache(qkv: torch.Tensor, pos: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor, hq: int, hkv: int, d: int,
               theta: float) -> None:
    rows = qkv.shape[0]
    call("rptc_rope_cache", qkv.device, ptr(qkv), _ld(qkv, qkv.shape[1]), ptr(pos), ptr(kcache), ptr(vcache), rows, hq, hkv, d,
         kcache.shape[1], theta)


def rope_cache_prompt(qkv: torch.Tensor, rows: int, tokens: int, kcache: torch.Tensor, vcache: torch.Tensor, hq: int, hkv: int, d: int,
                      theta: float) -> None:
    """RoPE of q (in place) and k, and the cache writes of k and v, for a whole prompt (rptc_rope_cache_prompt):
    qkv fp16 [rows * tokens, (hq + 2 hkv) d]."""
    call("rptc_rope_cache_prompt", qkv.device, ptr(qkv), _ld(qkv, qkv.shape[1]), rows, tokens, ptr(kcache), ptr(vcache), hq, hkv, d,
         kcache.shape[1], theta)


def rope_angles(tokens: int, theta: float, device) -> torch.Tensor:
    """Cosines and sines of positions 0 .. tokens-1 for 128-wide heads, fp32 [tokens, 64, 2] (rptc_rope_angles)."""
    out = torch.empty((tokens, 64, 2), dtype=torch.float32, device=device)
    call("rptc_rope_angles", out.device, ptr(out), tokens, theta)
    return out


def prompt_norm(y: torch.Tensor | None, signs_out: torch.Tensor | None, scale_out: float, h: torch.Tensor, w_norm: torch.Tensor, eps: float,
                signs_in: torch.Tensor | None, out: torch.Tensor) -> torch.Tensor:
    """h += output transform of the product y; out = input transform of rmsnorm(h), many rows (rptc_prompt_norm)."""
    rows, n = h.shape
    call("rptc_prompt_norm", h.device, ptr(y), 0 if y is None else _ld(y, n), ptr(signs_out), scale_out, ptr(h), _ld(h, n), ptr(w_norm), eps,
         ptr(signs_in), ptr(out), _ld(out, n), rows, n)
    return out


def prompt_qkv(qkv: torch.Tensor, signs_out: torch.Tensor | None, scale: float, rows: int, tokens: int, kcache: torch.Tensor,
               vcache: torch.Tensor, hq: int, hkv: int, angles: torch.Tensor) -> None:
    """Output transform of the fused qkv product + RoPE + cache writes for a whole prompt (rptc_prompt_qkv)."""
    call("rptc_prompt_qkv", qkv.device, ptr(qkv), _ld(qkv, qkv.shape[1]), ptr(signs_out), scale, rows, tokens, ptr(kcache), ptr(vcache), hq, hkv,
         kcache.shape[1], ptr(angles))


def attn_decode(qkv: torch.Tensor, pos: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor, out: torch.Tensor, hq: int,
                hkv: int, d: int, signs_in: torch.Tensor | None = None) -> torch.Tensor:
    rows = qkv.shape[0]
    call("rptc_attn_decode", qkv.device, ptr(qkv), _ld(qkv, qkv.shape[1]), ptr(pos), ptr(kcache), ptr(vcache), ptr(out),
         _ld(out, out.shape[1]), rows, hq, hkv, d, kcache.shape[1], d ** -0.5, ptr(signs_in))
    return out


def qkv_attn_decode(acc: torch.Tensor, signs_out: torch.Tensor | None, scale_out: float, pos: torch.Tensor, kcache: torch.Tensor,
                    vcache: torch.Tensor, out: torch.Tensor, heads: int, kv_heads: int, theta: float,
                    signs_in: torch.Tensor | None) -> torch.Tensor:
    """Output transform of the fused qkv layer + RoPE + KV append + attention (+ per-head input transform of the
    output projection) in one launch (rptc_qkv_attn_decode)."""
    rows = acc.shape[0]
    call("rptc_qkv_attn_decode", acc.device, ptr(acc), _ld(acc, acc.shape[1]), ptr(signs_out), scale_out, ptr(pos), ptr(kcache),
         ptr(vcache), ptr(out), _ld(out, out.shape[1]), rows, heads, kv_heads, kcache.shape[1], theta, ptr(signs_in))
    return out


def finish_norm_hadamard(acc: torch.Tensor | None, signs_out: torch.Tensor | None, scale_out: float, h: torch.Tensor,
                         w_norm: torch.Tensor, eps: float, signs_in: torch.Tensor | None, transform_in: bool,
                         out: torch.Tensor) -> torch.Tensor:
    """h += output transform of acc; out = input transform of rmsnorm(h) (rptc_finish_norm_hadamard)."""
    rows, n = h.shape
    call("rptc_finish_norm_hadamard", h.device, ptr(acc), 0 if acc is None else _ld(acc, n), ptr(signs_out), scale_out, ptr(h), _ld(h, n),
         ptr(w_norm), eps, ptr(signs_in), int(transform_in), ptr(out), _ld(out, n), rows, n)
    return out


def qkv_finish(acc: torch.Tensor, signs_out: torch.Tensor | None, scale: float, q_out: torch.Tensor, kcache: torch.Tensor,
               vcache: torch.Tensor, pos: torch.Tensor, hq: int, hkv: int, block: int, theta: float) -> None:
    """Output transform of the fused qkv layer + RoPE + KV-cache append (rptc_qkv_finish)."""
    rows = acc.shape[0]
    call("rptc_qkv_finish", acc.device, ptr(acc), _ld(acc, acc.shape[1]), ptr(signs_out), scale, ptr(q_out), _ld(q_out, q_out.shape[1]),
         ptr(kcache), ptr(vcache), ptr(pos), rows, hq, hkv, kcache.shape[1], block, theta)


def dense_gemv(W: torch.Tensor, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """y[b] = W x[b] for a dense fp16 W [m, n] (rptc_dense_gemv)."""
    squeeze = x.dim() == 1
    if squeeze:
        x = x.unsqueeze(0)
    m, n = W.shape
    if out is None:
        out = torch.empty((x.shape[0], m), dtype=torch.float16, device=x.device)
    o2 = out.unsqueeze(0) if out.dim() == 1 else out
    for b0 in range(0, x.shape[0], 16):                 # the kernel takes up to sixteen activation rows per launch
        xb, ob = x[b0:b0 + 16], o2[b0:b0 + 16]
        call("rptc_dense_gemv", W.device, ptr(W), W.stride(0), ptr(xb), _ld(xb, n), ptr(ob), _ld(ob, m), m, n, xb.shape[0])
    return out[0] if squeeze and out.dim() == 2 else out


def embed(table: torch.Tensor, ids: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    call("rptc_embed", table.device, ptr(table), ptr(ids), ptr(out), _ld(out, table.shape[1]), ids.shape[0], table.shape[1])
    return out


def embed_mailbox(table: torch.Tensor, slots: torch.Tensor, steps_done: torch.Tensor, ids: torch.Tensor, out: torch.Tensor,
                  timeout_ms: int = 2000) -> None:
    """Embedding rows of the ids the host posts in `slots` (pinned int64: sequence << 32 | id); waits for them, bounded
    (rptc_embed_mailbox)."""
    if not slots.is_pinned() or slots.dtype != torch.int64 or steps_done.dtype != torch.int32:
        raise RuntimeError("slots must be a pinned int64 host tensor and steps_done an int32 device tensor")
    call("rptc_embed_mailbox", table.device, ptr(table), ptr(slots), ptr(steps_done), ptr(ids), ptr(out), _ld(out, table.shape[1]),
         ids.shape[0], table.shape[1], table.shape[0], timeout_ms)


def next_token(logits: torch.Tensor, next_ids: torch.Tensor, ids: torch.Tensor | None = None, pos: torch.Tensor | None = None,
               mirror: torch.Tensor | None = None, steps_done: torch.Tensor | None = None) -> None:
    """Greedy choice + feedback + position bump in one launch (rptc_next_token).  `mirror`: pinned host int64."""
    rows, n = logits.shape
    if next_ids.dtype != torch.int64 or (mirror is not None and (mirror.dtype != torch.int64 or not mirror.is_pinned())):
        raise RuntimeError("next_ids must be int64 and mirror a pinned int64 host tensor")
    call("rptc_next_token", logits.device, ptr(logits), _ld(logits, n), rows, n, ptr(next_ids), ptr(ids), ptr(pos), ptr(mirror),
         ptr(steps_done))


# ---- prompts of different lengths, caches in 4 bits, log probabilities ---------------------------------------------------

def _on(device: torch.device, name: str, t: torch.Tensor, dtype, shape: tuple | None = None) -> None:
    """A tensor that a kernel reads as it is: dtype (or one of several), device, and contiguous in `shape` (None: any)."""
    if t.device != device or device.type != "cuda":
        raise RuntimeError(f"{name} must be a CUDA tensor on {device}")
    if t.dtype != dtype if isinstance(dtype, torch.dtype) else t.dtype not in dtype:
        raise RuntimeError(f"{name} must have dtype {dtype}, got {t.dtype}")
    if shape is not None and (tuple(t.shape) != shape or not t.is_contiguous()):
        raise RuntimeError(f"{name} must be contiguous {list(shape)}, got {list(t.shape)}")


def _answer(result, where: str):
    """What a native call gave: None where something is not as the kernels read it (checked and refused below the call)."""
    if type(result) is int:
        check(result, where)
    return result


def kv4_cache(rows: int, max_pos: int, kv_heads: int, device="cuda") -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """A layer's KV cache in 4 bits for 128-wide heads, empty: codes of k, (scale, minimum) of its groups of 32 values, the same
    for v (rptc_kv_cache); 160 bytes per position and kv head, where fp16 takes 512."""
    codes = lambda: torch.zeros((rows, kv_heads, max_pos, 64), dtype=torch.uint8, device=device)
    scales = lambda: torch.zeros((rows, kv_heads, max_pos, 4, 2), dtype=torch.float16, device=device)
    return codes(), scales(), codes(), scales()


def _kv_cache(cache, device: torch.device) -> _lib.KVCache:
    """(k, v) in fp16 [rows, max_pos, kv_heads, 128], or the four tensors of `kv4_cache`."""
    if len(cache) == 2:
        if cache[0].dim() != 4 or cache[0].shape[3] != 128:
            raise RuntimeError("an fp16 cache must be [rows, max_pos, kv_heads, 128]")
        for name, t in zip(("k cache", "v cache"), cache):
            _on(device, name, t, torch.float16, tuple(cache[0].shape))
        rows, max_pos, kv_heads, _ = cache[0].shape
        return _lib.KVCache(ptr(cache[0]), None, ptr(cache[1]), None, rows, max_pos, kv_heads, 16)
    if len(cache) != 4 or cache[0].dim() != 4:
        raise RuntimeError("a cache is (k, v) in fp16, or (k codes, k scales, v codes, v scales)")
    rows, kv_heads, max_pos, _ = cache[0].shape
    for i, name in enumerate(("k codes", "k scales", "v codes", "v scales")):
        _on(device, name, cache[i], torch.float16 if i % 2 else torch.uint8, (rows, kv_heads, max_pos) + ((4, 2) if i % 2 else (64,)))
    return _lib.KVCache(*[ptr(t) for t in cache], rows, max_pos, kv_heads, 4)


def _rows_of(name: str, t: torch.Tensor, device: torch.device, dtype, rows: int, width: int) -> None:
    _on(device, name, t, dtype)
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] < width or (t.stride(1) != 1 and t.shape[1] > 1):
        raise RuntimeError(f"{name} must be [{rows}, >= {width}] with unit column stride, got {list(t.shape)}")


def qkv_append(x: torch.Tensor, pos: torch.Tensor, angles: torch.Tensor, cache, heads: int, kv_heads: int, slots: torch.Tensor | None = None,
               signs_out: torch.Tensor | None = None, scale: float = 1.0, transform: bool = False, out: torch.Tensor | None = None,
               clear: bool = False) -> torch.Tensor:
    """Output side of a fused qkv layer for tokens of any sequences (rptc_qkv_append): x fp16 or fp32 [tokens, (heads + 2 kv_heads) * 128],
    y = x * scale (`transform`: s_out * H(x) * scale in blocks of 128); q and k rotated by `angles` (fp32 [>= max_pos, 64, 2]) of the token's
    position, k and v appended to `cache` (fp16 pair or `kv4_cache`) at [slots[t], pos[t]] (slots None: row t; pos -1: a token of no
    sequence, nothing is written).  Returns fp16 [tokens, (heads + 2 kv_heads) * 128] with q, k and v as finished; an `out` of fewer columns
    takes q alone.  `clear` zeroes an fp32 x.  `out` may be x itself; otherwise the two do not overlap."""
    done = _answer(native().qkv_append(x, pos, angles, cache, heads, kv_heads, slots, signs_out, scale, transform, out, clear), "rptc_qkv_append")
    if done is not None:
        return done
    device, width = x.device, (heads + 2 * kv_heads) * 128
    c = _kv_cache(cache, device)
    if heads <= 0 or kv_heads != c.kv_heads:
        raise RuntimeError(f"the cache has {c.kv_heads} kv heads, got heads {heads}, kv_heads {kv_heads}")
    if x.dim() != 2:
        raise RuntimeError("x must be [tokens, (heads + 2 kv_heads) * 128]")
    tokens = x.shape[0]
    _rows_of("x", x, device, (torch.float16, torch.float32), tokens, width)
    _on(device, "pos", pos, torch.int32, (tokens,))
    if slots is not None:
        _on(device, "slots", slots, torch.int32, (tokens,))
    if angles.dim() != 3 or angles.shape[0] < c.max_pos:
        raise RuntimeError(f"angles must be [>= {c.max_pos}, 64, 2]")
    _on(device, "angles", angles, torch.float32, (angles.shape[0], 64, 2))
    if signs_out is not None:
        _on(device, "signs_out", signs_out, torch.float16, (width,))
    if out is None:
        out = torch.empty((tokens, width), dtype=torch.float16, device=device)
    _rows_of("out", out, device, torch.float16, tokens, heads * 128)
    if tokens == 0:
        return out
    a = _lib.Append(ptr(x), _ld(x, width), ptr(signs_out), ptr(slots), ptr(pos), ptr(angles), ptr(out), _ld(out, out.shape[1]), tokens, heads,
                    int(x.dtype == torch.float32), int(clear), int(transform), int(out.shape[1] >= width), scale, c)
    call("rptc_qkv_append", device, ctypes.byref(a))
    return out


def kv4_values(cache, count: torch.Tensor, out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The values that the first count[r] (int32 [rows]) positions of row r of a 4-bit cache stand for, fp16 k and v [rows, max_pos, kv_heads,
    128]; other positions are left as they are (rptc_kv4_values)."""
    done = _answer(native().kv4_values(cache, count, out), "rptc_kv4_values")
    if done is not None:
        return done
    device = cache[0].device
    c = _kv_cache(cache, device)
    if c.bits != 4:
        raise RuntimeError("the cache must be one of kv4_cache")
    _on(device, "count", count, torch.int32, (c.rows,))
    shape = (c.rows, c.max_pos, c.kv_heads, 128)
    k, v = out if out is not None else (torch.empty(shape, dtype=torch.float16, device=device) for _ in range(2))
    for t in (k, v):
        _on(device, "out", t, torch.float16, shape)
    call("rptc_kv4_values", device, ctypes.byref(c), ptr(count), ptr(k), ptr(v))
    return k, v


def attn_decode_kv4(q: torch.Tensor, pos: torch.Tensor, cache, heads: int, out: torch.Tensor | None = None, scale: float | None = None,
                    signs_in: torch.Tensor | None = None) -> torch.Tensor:
    """Single-query attention over positions 0 .. pos[r] of row r of a 4-bit cache (rptc_attn_decode_kv4): q fp16 [rows, >= heads * 128] ->
    fp16 [rows, heads * 128].  pos -1: a row of no sequence, zeros.  signs_in: each head's output also goes through the 128-wide input
    transform of the output projection."""
    done = _answer(native().attn_decode_kv4(q, pos, cache, heads, out, scale, signs_in), "rptc_attn_decode_kv4")
    if done is not None:
        return done
    device = cache[0].device
    c = _kv_cache(cache, device)
    _rows_of("q", q, device, torch.float16, c.rows, heads * 128)
    _on(device, "pos", pos, torch.int32, (c.rows,))
    if out is None:
        out = torch.empty((c.rows, heads * 128), dtype=torch.float16, device=device)
    _rows_of("out", out, device, torch.float16, c.rows, heads * 128)
    if signs_in is not None:
        _on(device, "signs_in", signs_in, torch.float16, (heads * 128,))
    if c.rows == 0:
        return out
    need = lib().rptc_attn_decode_kv4_workspace_bytes(ctypes.byref(c), heads)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    call("rptc_attn_decode_kv4", device, ptr(q), _ld(q, q.shape[1]), ptr(pos), ctypes.byref(c), ptr(out), _ld(out, out.shape[1]), heads,
         128 ** -0.5 if scale is None else scale, ptr(signs_in), ptr(ws), need)
    return out


def attn_decode_kv4_joins(cache, heads: int) -> bool:
    """Whether `attn_decode_kv4` over this cache takes a workspace, and a second launch that joins the parts of a row in it."""
    return lib().rptc_attn_decode_kv4_workspace_bytes(ctypes.byref(_kv_cache(cache, cache[0].device)), heads) > 0


def attn_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, kv_first: torch.Tensor | None = None,
                kv_len: torch.Tensor | None = None, out: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Causal attention of packed prompts of different lengths (rptc_attn_prompt): q [tokens, heads, d], k and v [kv_tokens, kv_heads, d], fp16 or
    bf16, d 64 or 128, unit stride along d -> out [tokens, heads, d].  Sequence s has the queries starts[s] .. starts[s + 1] - 1 (int32
    [sequences + 1]) and, for prompts that continue a cached context, the keys kv_first[s] .. kv_first[s] + kv_len[s] - 1 (int32 [sequences]; None:
    its keys lie where its queries do); its last query sees all of them.  Rows of `out` behind the last sequence are left as they are."""
    done = _answer(native().attn_prompt(q, k, v, starts, kv_first, kv_len, out, scale), "rptc_attn_prompt")
    if done is not None:
        return done
    device = q.device
    for name, t in (("q", q), ("k", k), ("v", v)):
        _on(device, name, t, (torch.float16, torch.bfloat16))
        if t.dim() != 3 or t.dtype != q.dtype or t.shape[2] != q.shape[2] or t.stride(2) != 1:
            raise RuntimeError(f"{name} must be [rows, heads, d] of q's dtype and d with unit stride along d")
    if k.shape != v.shape:
        raise RuntimeError("k and v must have the same shape")
    tokens, heads, d = q.shape
    if starts.dim() != 1 or starts.shape[0] < 1:
        raise RuntimeError("starts must be int32 [sequences + 1]")
    n = starts.shape[0] - 1
    _on(device, "starts", starts, torch.int32, (n + 1,))
    if (kv_first is None) != (kv_len is None):
        raise RuntimeError("kv_first and kv_len go together")
    for name, t in (("kv_first", kv_first), ("kv_len", kv_len)):
        if t is not None:
            _on(device, name, t, torch.int32, (n,))
    if out is None:
        out = torch.empty((tokens, heads, d), dtype=q.dtype, device=device)
    _on(device, "out", out, q.dtype)
    if out.shape != q.shape or out.stride(2) != 1:
        raise RuntimeError("out must have q's shape and unit stride along d")
    if tokens == 0 or n == 0:
        return out
    if k.shape[0] == 0:
        raise RuntimeError("k and v must have at least one row")

    def strides(t):      # of an axis of one element any
        return (t.stride(0) if t.shape[0] > 1 else t.shape[1] * d, t.stride(1) if t.shape[1] > 1 else d)

    a = _lib.PromptAttention(ptr(q), ptr(k), ptr(v), ptr(out), ptr(starts), ptr(kv_first), ptr(kv_len), tokens, k.shape[0], n, *strides(q), *strides(k),
                             *strides(v), *strides(out), heads, k.shape[1], d, int(q.dtype == torch.bfloat16), d ** -0.5 if scale is None else scale)
    call("rptc_attn_prompt", device, ctypes.byref(a))
    return out


_LOGIT_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor | None = None, top: int = 0):
    """Log probabilities of given tokens, with entropy and alternatives (rptc_token_logprobs): logits fp16, bf16 or fp32 [rows, n], targets int64
    [rows] (-1: no token, 0) -> (logprob fp32 [rows] or None, entropy fp32 [rows], top_logprobs fp32 [rows, top], top_ids int64 [rows, top], the
    largest first, equal ones by their index).  -inf is a forbidden token."""
    done = _answer(native().token_logprobs(logits, targets, top), "rptc_token_logprobs")
    if done is not None:
        return done
    device = logits.device
    _on(device, "logits", logits, tuple(_LOGIT_TYPES))
    if logits.dim() != 2 or logits.shape[1] < 1 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise RuntimeError("logits must be [rows, n] with unit column stride")
    rows, n = logits.shape
    if not 0 <= top <= min(32, n):
        raise RuntimeError(f"top must be between 0 and {min(32, n)}, got {top}")
    if targets is not None:
        _on(device, "targets", targets, torch.int64, (rows,))
    f32 = dict(dtype=torch.float32, device=device)
    logprob, entropy = None if targets is None else torch.empty(rows, **f32), torch.empty(rows, **f32)
    best, ids = torch.empty((rows, top), **f32), torch.empty((rows, top), dtype=torch.int64, device=device)
    if rows == 0:
        return logprob, entropy, best, ids
    call("rptc_token_logprobs", device, ptr(logits), _LOGIT_TYPES[logits.dtype], _ld(logits, n), ptr(targets), ptr(logprob), ptr(entropy),
         ptr(best) if top else None, ptr(ids) if top else None, rows, n, top)
    return logprob, entropy, best, ids


def viterbi_encode(alphabet: torch.Tensor, pos_weight: torch.Tensor, samples: torch.Tensor, workspace_limit: int = 12 << 30):
    """Code-A trellis encoder on the GPU (rptc_viterbi_encode): samples fp32 [rows, n] -> (symbols int32 [rows, n],
    loss fp32 [rows])."""
    return viterbi_encode_banked(alphabet[None, :], pos_weight, samples, workspace_limit)


def quantiles(sorted_values: torch.Tensor, L: int) -> torch.Tensor:
    """2^L evenly spaced quantiles of each row of sorted fp32 values [banks, n] -> fp32 [banks, 2^L] (rptc_quantiles)."""
    _cuda_contig(sorted_values, "sorted_values", torch.float32)
    out = torch.empty((sorted_values.shape[0], 1 << L), dtype=torch.float32, device=sorted_values.device)
    call("rptc_quantiles", out.device, ptr(sorted_values), sorted_values.shape[0], sorted_values.shape[1], L, ptr(out))
    return out


def encoder_rows_at_once(L: int, n: int, sms: int, workspace_limit: int) -> int:
    """How many rows of n samples go through the encoder at once.  More than the kernel has in flight (one row per SM at L = 16, two
    at L = 15) only shorten the tail of the last ones, so beyond 4 GiB of survivor memory it is no more than those: 2.4 GB
    at L = 16 and n = 4096.  Whole sets of them, so that no launch ends with idle SMs."""
    fit = workspace_limit // lib().rptc_viterbi_workspace_bytes(1, n, L)
    flight = sms // 2 * 2 if L == 16 else 2 * sms
    most = max(flight, (4 << 30) // lib().rptc_viterbi_workspace_bytes(1, n, L))
    rows = max(1, min(65535, fit, most))
    return rows // flight * flight if rows >= flight else rows


def viterbi_encode_banked(alphabets: torch.Tensor, pos_weight: torch.Tensor, samples: torch.Tensor, workspace_limit: int = 12 << 30,
                          least_rows: int = 1):
    """The same for `alphabets` [banks, 2^L] whose banks own equal groups of consecutive rows of `samples`
    (rptc_viterbi_encode_rows).  Rows go through in batches whose survivor memory stays under `workspace_limit`
    (encoder_rows_at_once), and in smaller ones, down to `least_rows`, where the device has no room for that."""
    banks, M = alphabets.shape
    L = M.bit_length() - 1
    if M != 1 << L:
        raise RuntimeError("the alphabet must have 2^L entries")
    alphabets = alphabets.to(torch.float32).contiguous()
    pos_weight = pos_weight.to(torch.float32).contiguous()
    samples = samples.to(torch.float32).contiguous()
    rows, n = samples.shape
    if rows % banks:
        raise RuntimeError("the banks must hold equally many rows")
    symbols = torch.empty((rows, n), dtype=torch.int32, device=samples.device)
    loss = torch.empty(rows, dtype=torch.float32, device=samples.device)
    if rows == 0:
        return symbols, loss
    per_bank = rows // banks
    step = min(rows, encoder_rows_at_once(L, n, torch.cuda.get_device_properties(samples.device).multi_processor_count, workspace_limit))
    while True:
        need = lib().rptc_viterbi_workspace_bytes(step, n, L)
        try:
            ws = torch.empty(need, dtype=torch.uint8, device=samples.device)
            break
        except torch.OutOfMemoryError:
            if step <= least_rows:
                raise
            step = max(least_rows, step // 2)
    for r0 in range(0, rows, step):
        bank, inside = divmod(r0, per_bank)
        call("rptc_viterbi_encode_rows", samples.device, ptr(alphabets[bank:]), per_bank, inside, ptr(pos_weight), ptr(samples[r0:]), n,
             min(step, rows - r0), n, L, ptr(symbols[r0:]), n, ptr(loss[r0:]), ptr(ws), need)
    return symbols, loss


def device_status() -> None:
    """Raises if a kernel reported a timed-out wait since the last call."""
    check(lib().rptc_device_status(), "rptc_device_status")
