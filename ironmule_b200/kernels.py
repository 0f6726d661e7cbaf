"""Torch-facing wrappers of the libimspec kernels: device tensors in, device tensors out, the current CUDA
stream, no host synchronisation. PyTorch supplies memory and streams; the arithmetic is libimspec's.

Weights use MLX's affine 4-bit layout: `w` int32/uint32 [N, K/8] (8 codes per word, low nibble first),
`scales` and `biases` bf16 [N, K/64].

Kernels that reduce across CTAs borrow a zero-filled scratch buffer. Pass one explicitly (`ws=`, a uint8 CUDA
tensor from `workspace()`) where the call is captured in a CUDA graph or may overlap another call;
otherwise a shared per-device buffer is used.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
import threading

import torch

from . import _lib

_EPILOGUES = {"store": _lib.EPI_STORE, "residual": _lib.EPI_RESIDUAL, "swiglu": _lib.EPI_SWIGLU,
              "geglu": _lib.EPI_GEGLU}
_VARIANTS = {"auto": _lib.QGEMM_AUTO, "mma": _lib.QGEMM_MMA, "fma": _lib.QGEMM_FMA}


def _stream(device) -> int:
    """The handle of torch's current stream on the device (without building a Stream object where its index is known)."""
    index = getattr(device, "index", None)
    if not isinstance(index, int):  # "cuda", "cuda:0", torch.device("cuda")
        return torch.cuda.current_stream(device).cuda_stream
    return torch._C._cuda_getCurrentRawStream(index)


def _check(t: torch.Tensor, name: str, dtypes: tuple, device: torch.device | None = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path), got {t.device}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, expected one of {dtypes}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """A zero-filled scratch buffer of at least `nbytes` usable bytes (256-byte aligned inside)."""
    return torch.zeros(max(int(nbytes), 1 << 16) + 256, dtype=torch.uint8, device=device)


def _ws(buf: torch.Tensor, need: int) -> tuple[int, int]:
    ptr = buf.data_ptr()
    pad = (-ptr) % 256
    size = buf.numel() - pad
    if size < need:
        raise ValueError(f"workspace of {need} bytes needed, {size} given")
    return ptr + pad, size


class _Shared:
    """Per-(device, purpose) shared scratch for eager calls. The kernels leave counters at zero, so a buffer
    is reused as is; it grows by reallocation (never during CUDA graph capture: pass `ws=` there)."""

    buffers: dict[tuple, torch.Tensor] = {}
    lock = threading.Lock()

    @classmethod
    def get(cls, device: torch.device, need: int, purpose: str) -> torch.Tensor:
        key = (device.index, purpose)
        with cls.lock:
            buf = cls.buffers.get(key)
            if buf is None or buf.numel() - 256 < need:
                buf = workspace(need, device)
                cls.buffers[key] = buf
        return buf


def _ptr_or_none(t):
    return t.data_ptr() if t is not None else None


def _scratch(ws, device, need, purpose):
    if need == 0:
        return None, 0
    buf = ws if ws is not None else _Shared.get(device, need, purpose)
    return _ws(buf, need)


def qgemm_workspace_bytes(m: int, n: int, k: int) -> int:
    return int(_lib.load().im_qgemm_workspace_bytes(m, n, k))


def qgemm(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, *,
          epilogue: str = "store", residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
          variant: str = "auto", split_k: bool = True, ws: torch.Tensor | None = None,
          rows: int | None = None) -> torch.Tensor:
    """y[M, N] = x[M, K] . dequantize(w)[N, K]^T (bf16), or a fused epilogue of it. `rows` limits M to the
    first rows of x."""
    device = x.device
    _check(x, "x", (torch.bfloat16,))
    _check(w, "w", (torch.int32, torch.uint32), device)
    _check(scales, "scales", (torch.bfloat16,), device)
    _check(biases, "biases", (torch.bfloat16,), device)
    k = x.shape[-1]
    m = x.numel() // k if rows is None else rows
    n = w.shape[0]
    if w.shape[1] * 8 != k or scales.shape != (n, k // 64) or biases.shape != (n, k // 64):
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, w {tuple(w.shape)}, scales {tuple(scales.shape)}")
    epi = _EPILOGUES[epilogue]
    n_out = n // 2 if epi in (_lib.EPI_SWIGLU, _lib.EPI_GEGLU) else n
    if out is None:
        out = torch.empty((m, n_out), dtype=torch.bfloat16, device=device)
    elif out.dtype != torch.bfloat16 or out.device != device or out.numel() < m * n_out:
        raise ValueError("out must be a bf16 tensor on x's device with room for the result")
    res_ptr = None
    if epi == _lib.EPI_RESIDUAL:
        if residual is None or residual.dtype != torch.bfloat16 or residual.numel() < m * n:
            raise ValueError("the residual epilogue needs a bf16 `residual` of the output's size")
        res_ptr = residual.data_ptr()
    need = qgemm_workspace_bytes(m, n, k) if split_k else 0
    ws_ptr, ws_bytes = _scratch(ws, device, need, "qgemm")
    _lib.call("im_qgemm_w4g64_ex", w.data_ptr(), scales.data_ptr(), biases.data_ptr(), x.data_ptr(),
              out.data_ptr(), res_ptr, m, n, k, epi, _VARIANTS[variant], ws_ptr, ws_bytes, _stream(device))
    if rows is None and out.numel() == m * n_out:
        return out.view(*x.shape[:-1], n_out)
    return out


def argmax_workspace_bytes(rows: int, v: int) -> int:
    return int(_lib.load().im_argmax_workspace_bytes(rows, v))


def argmax_rows(logits: torch.Tensor, with_conf: bool = False, *, out: torch.Tensor | None = None,
                out_stride: int = 1, conf_out: torch.Tensor | None = None, ws: torch.Tensor | None = None,
                rows: int | None = None, ld: int | None = None):
    """(argmax int32, conf float32 or None) over the last axis of bf16 logits; row r starts at element r * ld
    (default: the vocabulary size); `out` may be a strided int32 buffer (row r written at out[r * out_stride])."""
    _check(logits, "logits", (torch.bfloat16,))
    device = logits.device
    v = logits.shape[-1]
    ld = v if ld is None else ld
    rows = logits.numel() // v if rows is None else rows
    if (rows - 1) * ld + v > logits.numel():
        raise ValueError("rows * ld exceed the logits buffer")
    idx = torch.empty(rows, dtype=torch.int32, device=device) if out is None else out
    conf = conf_out if conf_out is not None else (
        torch.empty(rows, dtype=torch.float32, device=device) if with_conf else None)
    ws_ptr, ws_bytes = _scratch(ws, device, argmax_workspace_bytes(rows, v), "argmax")
    _lib.call("im_argmax_rows", logits.data_ptr(), rows, v, ld, idx.data_ptr(), out_stride,
              conf.data_ptr() if conf is not None else None, ws_ptr, ws_bytes, _stream(device))
    return idx, conf


def verify_greedy(logits: torch.Tensor, drafts: torch.Tensor, *, b: int | None = None, k: int | None = None,
                  drafts_ld: int | None = None, tokens: torch.Tensor | None = None,
                  count: torch.Tensor | None = None, picks: torch.Tensor | None = None,
                  ws: torch.Tensor | None = None):
    """Greedy acceptance for B sequences with k drafts each: logits bf16 [B*(k+1), V], drafts int32 [B, k]
    (or a strided view: pass b, k, drafts_ld). Returns (tokens int32 [B, k+1] padded with -1, count int32 [B])."""
    _check(logits, "logits", (torch.bfloat16,))
    device = logits.device
    if drafts.dtype != torch.int32 or drafts.device != device:
        raise TypeError("drafts must be int32 on the logits' device")
    if b is None:
        b, k = drafts.shape
        drafts_ld = k
    v = logits.shape[-1]
    if logits.numel() < b * (k + 1) * v:
        raise ValueError("logits must hold B*(k+1) rows")
    tokens = torch.empty((b, k + 1), dtype=torch.int32, device=device) if tokens is None else tokens
    count = torch.empty(b, dtype=torch.int32, device=device) if count is None else count
    ws_ptr, ws_bytes = _scratch(ws, device, argmax_workspace_bytes(b * (k + 1), v), "argmax")
    _lib.call("im_verify_greedy", logits.data_ptr(), b, k, v, v, drafts.data_ptr(), drafts_ld, tokens.data_ptr(),
              count.data_ptr(), picks.data_ptr() if picks is not None else None, ws_ptr, ws_bytes,
              _stream(device))
    return tokens, count


def quantize(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """MLX-affine 4-bit, group-64 quantisation of bf16 w [N, K] on the device -> (wq int32 [N, K/8],
    scales bf16 [N, K/64], biases bf16 [N, K/64])."""
    _check(w, "w", (torch.bfloat16,))
    n, k = w.shape
    if k % 64:
        raise ValueError("K must be a multiple of 64")
    wq = torch.empty((n, k // 8), dtype=torch.int32, device=w.device)
    scales = torch.empty((n, k // 64), dtype=torch.bfloat16, device=w.device)
    biases = torch.empty((n, k // 64), dtype=torch.bfloat16, device=w.device)
    _lib.call("im_quantize_w4g64", w.data_ptr(), n, k, wq.data_ptr(), scales.data_ptr(), biases.data_ptr(),
              _stream(w.device))
    return wq, scales, biases


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, *, gemma: bool = False,
            out: torch.Tensor | None = None, rows: int | None = None, ldx: int | None = None) -> torch.Tensor:
    """RMSNorm of `rows` rows of x (row stride `ldx` elements; default: all rows, contiguous)."""
    _check(weight, "weight", (torch.bfloat16,), x.device)
    if x.dtype != torch.bfloat16 or x.device.type != "cuda":
        raise TypeError("x must be a bf16 CUDA tensor")
    h = weight.numel()
    ldx = h if ldx is None else ldx
    rows = x.numel() // h if rows is None else rows
    out = torch.empty((rows, h), dtype=torch.bfloat16, device=x.device) if out is None else out
    _lib.call("im_rmsnorm", x.data_ptr(), ldx, weight.data_ptr(), out.data_ptr(), rows, h, float(eps),
              int(gemma), _stream(x.device))
    return out


def rmsnorm_residual(y: torch.Tensor, weight: torch.Tensor | None, h: torch.Tensor, eps: float, *, gemma: bool = False,
                     rows: int | None = None, out_sq: torch.Tensor | None = None) -> torch.Tensor:
    """h += rmsnorm(y) * w' per row, in place (Gemma-3's output norms); out_sq gets the new rows' sums of squares."""
    hsz = h.shape[-1]
    m = h.numel() // hsz if rows is None else rows
    _lib.call("im_rmsnorm_residual", y.data_ptr(), _ptr_or_none(weight), h.data_ptr(), m, hsz, float(eps), int(gemma),
              _ptr_or_none(out_sq), _stream(h.device))
    return h


def qk_norm_rope_kv(qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor, inv_freq: torch.Tensor,
                    row_pos: torch.Tensor, row_slot: torch.Tensor, row_seq: torch.Tensor, page_table: torch.Tensor,
                    hq: int, hkv: int, d: int, eps: float, k_cache: torch.Tensor, v_cache: torch.Tensor, *,
                    gemma: bool = False, q_out: torch.Tensor | None = None, rows: int | None = None) -> torch.Tensor:
    m = qkv.shape[0] if rows is None else rows
    q_out = torch.empty((m, hq, d), dtype=torch.bfloat16, device=qkv.device) if q_out is None else q_out
    _lib.call("im_qk_norm_rope_kv", qkv.data_ptr(), q_norm.data_ptr(), k_norm.data_ptr(), inv_freq.data_ptr(),
              row_pos.data_ptr(), row_slot.data_ptr(), row_seq.data_ptr(), page_table.data_ptr(),
              page_table.shape[-1], m, hq, hkv, d, float(eps), int(gemma), q_out.data_ptr(), k_cache.data_ptr(),
              v_cache.data_ptr(), _stream(qkv.device))
    return q_out


def embed(tokens: torch.Tensor, wq: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, *,
          mult: float = 1.0, out: torch.Tensor | None = None, rows: int | None = None,
          stride: int = 1, out_sq: torch.Tensor | None = None) -> torch.Tensor:
    """Rows tokens[0], tokens[stride], ... of the 4-bit table, dequantised (bf16 [rows, H])."""
    if tokens.dtype != torch.int32 or tokens.device.type != "cuda":
        raise TypeError("tokens must be an int32 CUDA tensor")
    v, h = wq.shape[0], wq.shape[1] * 8
    m = tokens.numel() if rows is None else rows
    out = torch.empty((m, h), dtype=torch.bfloat16, device=tokens.device) if out is None else out
    _lib.call("im_embed_w4g64", tokens.data_ptr(), stride, wq.data_ptr(), scales.data_ptr(), biases.data_ptr(), m,
              v, h, float(mult), out.data_ptr(), _ptr_or_none(out_sq), _stream(tokens.device))
    return out


def attention_workspace_bytes(b: int, rows: int, hq: int, hkv: int, d: int, max_kv_len: int, kpc: int) -> int:
    return int(_lib.load().im_attention_workspace_bytes(b, rows, hq, hkv, d, max_kv_len, kpc))


def attention_tune(waves: int) -> None:
    """Waves of resident CTAs the attention launch aims for (scheduling only; results do not change)."""
    _lib.call("im_attention_tune", int(waves))


def attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
              seq_rows: torch.Tensor, row_slot: torch.Tensor, *, max_rows_per_seq: int, max_kv_len: int,
              scale: float, keys_per_split: int = 64, window: int = 0, tree_mask: torch.Tensor | None = None,
              tree_base: torch.Tensor | None = None, out: torch.Tensor | None = None, rows: int | None = None,
              ws: torch.Tensor | None = None, seq_slot: torch.Tensor | None = None) -> torch.Tensor:
    """Paged verification attention; q [M, Hq, D] -> out [M, Hq, D] (bf16)."""
    hq, d = q.shape[-2], q.shape[-1]
    m = q.shape[0] if rows is None else rows
    hkv = k_cache.shape[-3]
    b = seq_rows.numel() - 1
    out = torch.empty((m, hq, d), dtype=torch.bfloat16, device=q.device) if out is None else out
    need = attention_workspace_bytes(b, max_rows_per_seq, hq, hkv, d, max_kv_len, keys_per_split)
    if need == 0:
        raise ValueError("attention shape not supported")
    ws_ptr, ws_bytes = _scratch(ws, q.device, need, "attention")
    _lib.call("im_attention_paged", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(),
              page_table.shape[-1], seq_rows.data_ptr(), _ptr_or_none(seq_slot), row_slot.data_ptr(),
              tree_mask.data_ptr() if tree_mask is not None else None,
              tree_base.data_ptr() if tree_base is not None else None, b, max_rows_per_seq, hq, hkv, d, max_kv_len,
              keys_per_split, window, float(scale), out.data_ptr(), ws_ptr, ws_bytes, _stream(q.device))
    return out


def attention_qkv(qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor, inv_freq: torch.Tensor,
                  row_pos: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                  seq_rows: torch.Tensor, row_slot: torch.Tensor, *, hq: int, hkv: int, d: int, eps: float,
                  max_rows_per_seq: int, max_kv_len: int, scale: float, gemma: bool = False,
                  keys_per_split: int = 64, window: int = 0, tree_mask: torch.Tensor | None = None,
                  tree_base: torch.Tensor | None = None, out: torch.Tensor | None = None, rows: int | None = None,
                  ws: torch.Tensor | None = None, seq_slot: torch.Tensor | None = None,
                  defer: bool = False) -> torch.Tensor | None:
    """Attention from the packed qkv projection rows [M, (Hq + 2 Hkv) D]: q/k RMSNorm + RoPE and the K/V cache
    write happen inside the kernel; returns out [M, Hq, D] (bf16). defer: only the split partials are written
    (into ws), for qgemm_packed_attn to merge; returns None."""
    if qkv.dtype != torch.bfloat16 or not qkv.is_contiguous():
        raise TypeError("qkv must be a contiguous bf16 tensor")
    m = qkv.shape[0] if rows is None else rows
    b = seq_rows.numel() - 1
    if defer and ws is None:
        raise ValueError("a deferred merge needs the workspace its consumer reads")
    if not defer:
        out = torch.empty((m, hq, d), dtype=torch.bfloat16, device=qkv.device) if out is None else out
    need = attention_workspace_bytes(b, max_rows_per_seq, hq, hkv, d, max_kv_len, keys_per_split)
    if need == 0:
        raise ValueError("attention shape not supported")
    ws_ptr, ws_bytes = _scratch(ws, qkv.device, need, "attention")
    _lib.call("im_attention_qkv_paged", qkv.data_ptr(), q_norm.data_ptr(), k_norm.data_ptr(), inv_freq.data_ptr(),
              row_pos.data_ptr(), float(eps), int(gemma), k_cache.data_ptr(), v_cache.data_ptr(),
              page_table.data_ptr(), page_table.shape[-1], seq_rows.data_ptr(), _ptr_or_none(seq_slot),
              row_slot.data_ptr(), _ptr_or_none(tree_mask), _ptr_or_none(tree_base), b, max_rows_per_seq, hq, hkv,
              d, max_kv_len, keys_per_split, window, float(scale), None if defer else out.data_ptr(), ws_ptr,
              ws_bytes, _stream(qkv.device))
    return None if defer else out


def spec_prepare(hist, n, target, b: int, k: int, slot_cap: int, d0_tok, d0_pos, d_pos, v_tok, v_pos) -> None:
    _lib.call("im_spec_prepare", hist.data_ptr(), hist.shape[-1], n.data_ptr(), target.data_ptr(), b, k, slot_cap,
              d0_tok.data_ptr(), d0_pos.data_ptr(), d_pos.data_ptr() if d_pos is not None else None,
              v_tok.data_ptr(), v_pos.data_ptr(), _stream(hist.device))


def spec_commit(hist, n, target, b: int, k: int, out_tokens, out_count, stats=None) -> None:
    _lib.call("im_spec_commit", hist.data_ptr(), hist.shape[-1], n.data_ptr(), target.data_ptr(), b, k,
              out_tokens.data_ptr(), out_count.data_ptr(), stats.data_ptr() if stats is not None else None,
              _stream(hist.device))


def sampling_workspace_bytes(rows: int) -> int:
    return int(_lib.load().im_sampling_workspace_bytes(rows))


def sample_rows(logits: torch.Tensor, temperature: float, top_p: float, seed: int, offset: int = 0, *,
                offset_dev: torch.Tensor | None = None, streams: torch.Tensor | None = None, draw: int = 0,
                out: torch.Tensor | None = None, out_stride: int = 1, rows: int | None = None,
                ws: torch.Tensor | None = None) -> torch.Tensor:
    """One token per row from softmax(logits / T) restricted to top-p, on the Philox stream."""
    _check(logits, "logits", (torch.bfloat16,))
    v = logits.shape[-1]
    rows = logits.numel() // v if rows is None else rows
    out = torch.empty(rows, dtype=torch.int32, device=logits.device) if out is None else out
    ws_ptr, ws_bytes = _scratch(ws, logits.device, sampling_workspace_bytes(rows), "sampling")
    _lib.call("im_sample_rows", logits.data_ptr(), rows, v, v, float(temperature), float(top_p), int(seed),
              int(offset), _ptr_or_none(offset_dev), _ptr_or_none(streams), int(draw), out.data_ptr(), out_stride,
              ws_ptr, ws_bytes, _stream(logits.device))
    return out


def accept_stochastic(target_logits: torch.Tensor, draft_logits: torch.Tensor, drafts: torch.Tensor, *, b: int,
                      k: int, drafts_ld: int, temperature: float, top_p: float, seed: int, offset: int = 0,
                      offset_dev: torch.Tensor | None = None, tokens: torch.Tensor | None = None,
                      count: torch.Tensor | None = None, ratios: torch.Tensor | None = None,
                      ws: torch.Tensor | None = None):
    """p/q rejection sampling: target_logits [B, k+1, V], draft_logits [k, B, V] -> (tokens [B, k+1], count [B])."""
    _check(target_logits, "target_logits", (torch.bfloat16,))
    _check(draft_logits, "draft_logits", (torch.bfloat16,), target_logits.device)
    device = target_logits.device
    v = target_logits.shape[-1]
    tokens = torch.empty((b, k + 1), dtype=torch.int32, device=device) if tokens is None else tokens
    count = torch.empty(b, dtype=torch.int32, device=device) if count is None else count
    ws_ptr, ws_bytes = _scratch(ws, device, sampling_workspace_bytes(b * (2 * k + 1)), "sampling")
    _lib.call("im_accept_stochastic", target_logits.data_ptr(), draft_logits.data_ptr(), b, k, v, v,
              drafts.data_ptr(), drafts_ld, float(temperature), float(top_p), int(seed), int(offset),
              _ptr_or_none(offset_dev), tokens.data_ptr(), count.data_ptr(), _ptr_or_none(ratios), ws_ptr,
              ws_bytes, _stream(device))
    return tokens, count


def topk_workspace_bytes(rows: int, v: int, k: int) -> int:
    return int(_lib.load().im_topk_workspace_bytes(rows, v, k))


def topk_rows(logits: torch.Tensor, k: int, *, rows: int | None = None, ld: int | None = None,
              out: torch.Tensor | None = None, out_stride: int | None = None,
              ws: torch.Tensor | None = None) -> torch.Tensor:
    """The k largest entries of each row (indices, largest first, ties to the lower index)."""
    _check(logits, "logits", (torch.bfloat16,))
    v = logits.shape[-1]
    ld = v if ld is None else ld
    rows = logits.numel() // v if rows is None else rows
    out_stride = k if out_stride is None else out_stride
    out = torch.empty((rows, k), dtype=torch.int32, device=logits.device) if out is None else out
    ws_ptr, ws_bytes = _scratch(ws, logits.device, topk_workspace_bytes(rows, v, k), "topk")
    _lib.call("im_topk_rows", logits.data_ptr(), rows, v, ld, k, out.data_ptr(), out_stride, ws_ptr, ws_bytes,
              _stream(logits.device))
    return out


def _branch(branch) -> ctypes.Array:
    return (ctypes.c_int32 * len(branch))(*branch)


def tree_prepare(hist, n, branch, slot_cap: int, d0_tok, d0_pos, v_tok, v_pos, v_slot, v_mask, tree_base) -> None:
    _lib.call("im_tree_prepare", hist.data_ptr(), hist.shape[-1], n.data_ptr(), n.numel(), _branch(branch),
              len(branch), slot_cap, d0_tok.data_ptr(), d0_pos.data_ptr(), v_tok.data_ptr(), v_pos.data_ptr(),
              v_slot.data_ptr(), v_mask.data_ptr(), tree_base.data_ptr(), _stream(hist.device))


def tree_accept(argmax, v_tok, b: int, branch, out_tokens, out_count, acc_node) -> None:
    _lib.call("im_tree_accept", argmax.data_ptr(), v_tok.data_ptr(), b, _branch(branch), len(branch),
              out_tokens.data_ptr(), out_count.data_ptr(), acc_node.data_ptr(), _stream(argmax.device))


def tree_compact(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table, tree_base, acc_node, levels: int,
                 max_depth: int, b: int) -> None:
    """k_cache / v_cache [layers, pages, Hkv, 16, D]."""
    layers, _, hkv, _, d = k_cache.shape
    _lib.call("im_tree_compact", k_cache.data_ptr(), v_cache.data_ptr(), layers, k_cache.stride(0),
              page_table.data_ptr(), page_table.shape[-1], tree_base.data_ptr(), acc_node.data_ptr(), levels,
              max_depth, b, hkv, d, _stream(k_cache.device))


def philox(seed: int, offset: int, stream_id: int, n: int, device) -> torch.Tensor:
    out = torch.empty((n, 4), dtype=torch.int32, device=device)
    _lib.call("im_philox4x32_10", int(seed), int(offset), int(stream_id), int(n), out.data_ptr(), _stream(device))
    return out


# ---- packed weights (the engine's resident format) ------------------------------------------------------
class Packed:
    """A 4-bit projection repacked into MMA-fragment order (im_qgemm_pack_w4g64): n rows, k inputs."""

    def __init__(self, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor):
        _check(w, "w", (torch.int32, torch.uint32))
        self.n, self.k = int(w.shape[0]), int(w.shape[1]) * 8
        nbytes = int(_lib.load().im_qgemm_packed_bytes(self.n, self.k))
        self.data = torch.empty(nbytes, dtype=torch.uint8, device=w.device)
        _lib.call("im_qgemm_pack_w4g64", w.data_ptr(), scales.data_ptr(), biases.data_ptr(), self.n, self.k,
                  self.data.data_ptr(), _stream(w.device))

    @property
    def tiles(self) -> int:
        return (self.n + 31) // 32


def set_launch_overlap(on: bool) -> bool:
    """Programmatic dependent launch of the decode-path kernels on (default) or off; returns the previous
    setting. Results are bit-identical either way."""
    return bool(_lib.load().im_set_launch_overlap(int(bool(on))))


def set_wait_limit(ns: int) -> int:
    """Nanoseconds after which a bounded wait of the tensor-core products (packed qGEMM, products by expert) gives up (a
    second by default); returns the previous limit. Calls made from now on, captured graphs not."""
    return int(_lib.load().im_set_wait_limit(ns))


def qgemm_packed_workspace_bytes(m: int, n: int, k: int) -> int:
    return int(_lib.load().im_qgemm_packed_workspace_bytes(m, n, k))


def qgemm_packed_status(ws: torch.Tensor) -> int:
    """The error word of a workspace last used by a call of more than 32 rows (0: every wait completed); waits for the
    device."""
    ptr, _ = _ws(ws, 1 << 16)
    with torch.cuda.device(ws.device):
        return int(_lib.load().im_qgemm_packed_status(ptr))


def qgemm_packed_path(path: int) -> None:
    """0: automatic (default); 1: warp MMA always; 2: tcgen05 tensor cores always. Every choice gives the same
    bits."""
    _lib.call("im_qgemm_packed_path", int(path))


def qgemm_packed_cluster(on: bool) -> None:
    """Split-K partials of the warp-MMA kernel summed inside a thread-block cluster (True, default) or through
    the workspace and a global counter (False). Both give the same bits."""
    _lib.call("im_qgemm_packed_cluster", int(bool(on)))


def qgemm_packed_tune(split_override: int = 0, target_ctas: int = 592, max_split: int = 16) -> None:
    """The K-split policy (process-wide; changes workspace sizes)."""
    _lib.call("im_qgemm_packed_tune", split_override, target_ctas, max_split)


def qgemm_packed(x: torch.Tensor, p: Packed, *, epilogue: str = "store", residual: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, rows: int | None = None, norm_sq: torch.Tensor | None = None,
                 norm_parts: int = 0, norm_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 gemma_norm: bool = False, out_sq: torch.Tensor | None = None, sq_ld: int = 0,
                 ws: torch.Tensor | None = None) -> torch.Tensor:
    """y = x . W^T over packed weights, with an optional fused RMSNorm prologue (norm_sq/norm_weight) and
    per-tile sums of squares of the output (out_sq)."""
    device = x.device
    if x.dtype != torch.bfloat16 or device.type != "cuda" or not x.is_contiguous():
        raise TypeError("x must be a contiguous bf16 CUDA tensor")
    k = x.shape[-1]
    if k != p.k:
        raise ValueError(f"x has K={k}, the weights {p.k}")
    m = x.numel() // k if rows is None else rows
    epi = _EPILOGUES[epilogue]
    n_out = p.n // 2 if epi in (_lib.EPI_SWIGLU, _lib.EPI_GEGLU) else p.n
    out = torch.empty((m, n_out), dtype=torch.bfloat16, device=device) if out is None else out
    ws_ptr, ws_bytes = _scratch(ws, device, qgemm_packed_workspace_bytes(m, p.n, p.k), "qgemm_packed")
    _lib.call("im_qgemm_packed", p.data.data_ptr(), x.data_ptr(), out.data_ptr(), _ptr_or_none(residual), m, p.n, p.k,
              epi, _ptr_or_none(norm_sq), norm_parts, _ptr_or_none(norm_weight), float(eps), int(gemma_norm),
              _ptr_or_none(out_sq), sq_ld, ws_ptr, ws_bytes, _stream(device))
    return out


def qgemm_packed_attn_rows(n: int, k: int) -> int:
    """The most rows qgemm_packed_attn takes for an [n, k] projection (0: none)."""
    return int(_lib.load().im_qgemm_packed_attn_rows(n, k))


def qgemm_packed_attn(attn_ws: torch.Tensor, p: Packed, seq_rows: torch.Tensor, row_slot: torch.Tensor, *,
                      residual: torch.Tensor, out: torch.Tensor, rows: int, max_rows_per_seq: int, hq: int, hkv: int,
                      d: int, max_kv_len: int, keys_per_split: int, out_sq: torch.Tensor | None = None,
                      sq_ld: int = 0, ws: torch.Tensor | None = None) -> torch.Tensor:
    """The o-projection with a residual epilogue whose input is the attention output merged, in its prologue,
    from the split partials that attention_qkv(..., defer=True) left in attn_ws (the same bits as merging them
    in the attention and projecting its output). Takes at most qgemm_packed_attn_rows(p.n, p.k) rows."""
    device = residual.device
    b = seq_rows.numel() - 1
    ws_ptr, ws_bytes = _scratch(ws, device, qgemm_packed_workspace_bytes(rows, p.n, p.k), "qgemm_packed")
    _lib.call("im_qgemm_packed_attn", p.data.data_ptr(), attn_ws.data_ptr(), seq_rows.data_ptr(), row_slot.data_ptr(),
              b, max_rows_per_seq, hq, hkv, d, max_kv_len, keys_per_split, out.data_ptr(), residual.data_ptr(), rows,
              p.n, p.k, _ptr_or_none(out_sq), sq_ld, ws_ptr, ws_bytes, _stream(device))
    return out


# ---- mixture-of-experts blocks ------------------------------------------------------------------------------
_SCORING = {"softmax": _lib.MOE_SOFTMAX, "sigmoid": _lib.MOE_SIGMOID}


class Experts:
    """E 4-bit matrices [N, K] of one shape, repacked once for the products by expert: w int32 [E, N, K/8], scales and
    biases bf16 [E, N, K/64] (MLX's layout of stacked experts)."""

    def __init__(self, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor):
        _check(w, "w", (torch.int32, torch.uint32))
        _check(scales, "scales", (torch.bfloat16,), w.device)
        _check(biases, "biases", (torch.bfloat16,), w.device)
        if w.dim() != 3:
            raise ValueError(f"w must be [E, N, K/8], got {tuple(w.shape)}")
        self.e, self.n, self.k = int(w.shape[0]), int(w.shape[1]), int(w.shape[2]) * 8
        if scales.shape != (self.e, self.n, self.k // 64) or biases.shape != scales.shape:
            raise ValueError(f"shape mismatch: w {tuple(w.shape)}, scales {tuple(scales.shape)}, "
                             f"biases {tuple(biases.shape)}")
        nbytes = int(_lib.load().im_moe_packed_bytes(self.e, self.n, self.k))
        self.data = torch.empty(nbytes, dtype=torch.uint8, device=w.device)
        _lib.call("im_moe_pack_w4g64", w.data_ptr(), scales.data_ptr(), biases.data_ptr(), self.e, self.n, self.k,
                  self.data.data_ptr(), _stream(w.device))

    @classmethod
    def gate_up(cls, gate: tuple, up: tuple) -> "Experts":
        """The first product of a gated MLP: gate and up as (w, scales, biases) of [E, I, K], interleaved in 16-row
        blocks so that one tile holds both halves of its outputs."""
        def weave(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
            e, i, c = g.shape
            if u.shape != g.shape or i % 16:
                raise ValueError("gate and up must have one shape, the intermediate size a multiple of 16")
            return torch.stack([g.view(e, i // 16, 16, c), u.view(e, i // 16, 16, c)], dim=2).reshape(e, 2 * i, c)

        return cls(*(weave(g.contiguous(), u.contiguous()) for g, u in zip(gate, up)))


class Routing:
    """What moe_route found, in one int32 buffer: per row and place the expert (`ids` int32 [M, k], -1: none) and its
    weight (`weights` float32 [M, k]); the pairs m * k + j sorted by expert (`pairs` int32 [M * k]), where each expert's
    begin (`offsets` int32 [E + 2]; the last bucket holds the places without an expert), and the products' work items.
    The tensors are views made when they are asked for."""

    __slots__ = ("buf", "rows", "experts", "top_k", "plan_bytes", "error")

    def __init__(self, rows: int, experts: int, top_k: int, device: torch.device, error: torch.Tensor | None = None):
        self.rows, self.experts, self.top_k, self.error = rows, experts, top_k, error
        self.plan_bytes = _plan_bytes(rows, experts, top_k)
        self.buf = torch.empty(self._plan_at + self.plan_bytes // 4, dtype=torch.int32, device=device)

    @property
    def _plan_at(self) -> int:  # 16-byte aligned, after ids, weights, pairs and offsets
        return (3 * self.rows * self.top_k + self.experts + 2 + 3) // 4 * 4

    @property
    def ids(self) -> torch.Tensor:
        return torch.as_strided(self.buf, (self.rows, self.top_k), (self.top_k, 1), 0)

    @property
    def weights(self) -> torch.Tensor:
        return torch.as_strided(self.buf.view(torch.float32), (self.rows, self.top_k), (self.top_k, 1),
                                self.rows * self.top_k)

    @property
    def pairs(self) -> torch.Tensor:
        n = self.rows * self.top_k
        return torch.as_strided(self.buf, (n,), (1,), 2 * n)

    @property
    def offsets(self) -> torch.Tensor:
        return torch.as_strided(self.buf, (self.experts + 2,), (1,), 3 * self.rows * self.top_k)

    @property
    def _pairs_ptr(self) -> int:
        return self.buf.data_ptr() + 8 * self.rows * self.top_k

    @property
    def _plan_ptr(self) -> int:
        return self.buf.data_ptr() + 4 * self._plan_at

    def status(self) -> int:
        """The error word of the products that used this routing (0: every bounded wait completed); waits for the
        device, so for products on any stream."""
        with torch.cuda.device(self.buf.device):
            return int(_lib.load().im_moe_status(self._plan_ptr))


@functools.lru_cache(maxsize=4096)
def _plan_bytes(m: int, e: int, k: int) -> int:
    return int(_lib.load().im_moe_plan_bytes(m, e, k))


@functools.lru_cache(maxsize=4096)
def _grouped_workspace(m: int, e: int, k: int, kdim: int) -> int:
    return int(_lib.load().im_moe_grouped_workspace_bytes(m, e, k, kdim))


@functools.lru_cache(maxsize=4096)
def _mlp_workspace(m: int, e: int, k: int, h: int, inter: int) -> int:
    return int(_lib.load().im_moe_mlp_workspace_bytes(m, e, k, h, inter))


def moe_route(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax", normalise: bool = True,
              scale: float = 1.0, bias: torch.Tensor | None = None, bias_on: str = "logit",
              rows: int | None = None, error: torch.Tensor | None = None) -> Routing:
    """Choose top_k experts for each of the first `rows` rows of logits [M, E] (bf16 or float32): the largest
    logit + bias, ties to the lower expert; -inf or NaN closes an expert to a row. bias_on="score" chooses by
    sigmoid(logit) + bias or softmax(logits) + bias instead, what the correction bias of a load-balanced router is
    trained for. The bias only chooses: weights are the unbiased scores. `error` (one int32) is set to 1 when a bounded
    wait of a product of this routing runs out: a word that a program keeps for many calls."""
    _check(logits, "logits", (torch.bfloat16, torch.float32))
    if logits.dim() != 2:
        raise ValueError(f"logits must be [M, E], got {tuple(logits.shape)}")
    if scoring not in _SCORING:
        raise ValueError(f"scoring {scoring!r}: softmax or sigmoid")
    if bias_on not in ("logit", "score"):
        raise ValueError(f"bias_on {bias_on!r}: logit or score")
    how = _SCORING[scoring] + (_lib.MOE_BIAS_ON_SCORE if bias is not None and bias_on == "score" else 0)
    device, e = logits.device, logits.shape[1]
    m = logits.shape[0] if rows is None else rows
    if not 0 <= m <= logits.shape[0]:
        raise ValueError(f"{m} rows of {logits.shape[0]}")
    if bias is not None:
        _check(bias, "bias", (torch.float32,), device)
        if bias.shape != (e,):
            raise ValueError(f"bias must be [{e}], got {tuple(bias.shape)}")
    if not 1 <= top_k <= e:
        raise ValueError(f"top_k {top_k} of {e} experts")
    if error is not None:
        _check(error, "error", (torch.int32,), device)
        if error.numel() != 1:
            raise ValueError(f"error must be one element, got {tuple(error.shape)}")
    r = Routing(m, e, top_k, device, error)
    base, n = r.buf.data_ptr(), 4 * m * top_k
    _lib.call("im_moe_route_ex", logits.data_ptr(), int(logits.dtype == torch.float32), m, e, e, _ptr_or_none(bias), top_k,
              how, int(normalise), float(scale), base, base + n, base + 3 * n, base + 2 * n,
              r._plan_ptr, r.plan_bytes, _ptr_or_none(error), _stream(device))
    return r


def _moe_rows(x: torch.Tensor, experts: Experts, routing: Routing) -> bool:
    """Check x against the routing and the weights; whether x holds a row per pair ([M, k, K]) or per row ([M, K])."""
    _check(x, "x", (torch.bfloat16,), experts.data.device)
    if routing.buf.device != x.device:
        raise ValueError(f"the routing is on {routing.buf.device}, x on {x.device}")
    if x.shape[-1] != experts.k:
        raise ValueError(f"x has K={x.shape[-1]}, the experts {experts.k}")
    if experts.e != routing.experts:
        raise ValueError(f"{experts.e} experts, the routing is over {routing.experts}")
    by_pair = x.dim() == 3
    if x.shape[:-1] != ((routing.rows, routing.top_k) if by_pair else (routing.rows,)):
        raise ValueError(f"x {tuple(x.shape)} does not match a routing of {routing.rows} rows, {routing.top_k} places")
    return by_pair


def _moe_out(out: torch.Tensor | None, shape: tuple, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return like.new_empty(shape)
    _check(out, "out", (torch.bfloat16,), like.device)
    if out.shape != shape:
        raise ValueError(f"out must be {shape}, got {tuple(out.shape)}")
    return out


def grouped_qgemm(x: torch.Tensor, experts: Experts, routing: Routing, *,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """y[m, j] = W[ids[m, j]] x[m] for x [M, K], or W[ids[m, j]] x[m, j] for x [M, k, K]; bf16 [M, k, N], zero for
    places without an expert."""
    by_pair = _moe_rows(x, experts, routing)
    out = _moe_out(out, (routing.rows, routing.top_k, experts.n), x)
    need = _grouped_workspace(routing.rows, experts.e, routing.top_k, experts.k)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    _lib.call("im_moe_grouped_qgemm", experts.data.data_ptr(), x.data_ptr(), out.data_ptr(), routing.rows, experts.e,
              routing.top_k, experts.n, experts.k, int(by_pair), routing._pairs_ptr, routing._plan_ptr,
              routing.plan_bytes, ws.data_ptr(), need, _stream(x.device))
    return out


def moe_mlp(x: torch.Tensor, gate_up: Experts, down: Experts, routing: Routing, *, activation: str = "swiglu",
            out: torch.Tensor | None = None) -> torch.Tensor:
    """y[m, j] = D (act(G x[m]) * (U x[m])) with the matrices of expert ids[m, j]; act "swiglu" or "geglu"; bf16
    [M, k, H], zero for places without an expert. `gate_up` is Experts.gate_up's."""
    if _moe_rows(x, gate_up, routing):
        raise ValueError("x must be [M, H]")
    if activation not in ("swiglu", "geglu"):
        raise ValueError(f"activation {activation!r}: swiglu or geglu")
    if gate_up.n % 2:
        raise ValueError(f"gate_up has {gate_up.n} rows: gate and up rows come in pairs (Experts.gate_up)")
    h, inter = gate_up.k, gate_up.n // 2
    if (down.e, down.n, down.k) != (gate_up.e, h, inter) or down.data.device != x.device:
        raise ValueError(f"down is {down.e} x [{down.n}, {down.k}], expected {gate_up.e} x [{h}, {inter}]")
    out = _moe_out(out, (routing.rows, routing.top_k, h), x)
    need = _mlp_workspace(routing.rows, gate_up.e, routing.top_k, h, inter)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    _lib.call("im_moe_mlp", gate_up.data.data_ptr(), down.data.data_ptr(), x.data_ptr(), out.data_ptr(), routing.rows,
              gate_up.e, routing.top_k, h, inter, _EPILOGUES[activation], routing._pairs_ptr, routing._plan_ptr,
              routing.plan_bytes, ws.data_ptr(), need, _stream(x.device))
    return out


def _check_vector(t: torch.Tensor, name: str, n: int, device: torch.device) -> None:
    _check(t, name, (torch.bfloat16,), device)
    if t.shape != (n,):
        raise ValueError(f"{name} must be [{n}], got {tuple(t.shape)}")


def block_residual(y: torch.Tensor, h: torch.Tensor, eps: float, *, weights: torch.Tensor | None = None,
                   post_norm: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                   residual_scale: float = 1.0, next_norm: torch.Tensor | None = None, gemma: bool = False,
                   out: torch.Tensor | None = None, out_sq: torch.Tensor | None = None):
    """(h', z): a block's output joins the residual stream and the next block's input is normalised, in one pass.
    b = sum_j weights[m, j] y[m, j] (y [M, k, H] with weights float32 [M, k]; or y [M, H]); with post_norm its RMSNorm;
    h' = residual_scale * h + gate * b (gate bf16 [H], [M, 1] or [M, H]); z = RMSNorm(h') with next_norm, else None.
    `out` may be h. out_sq (float32 [M]) gets the sums of squares of the rounded h' rows."""
    _check(h, "h", (torch.bfloat16,))
    device = h.device
    _check(y, "y", (torch.bfloat16,), device)
    if h.dim() != 2:
        raise ValueError(f"h must be [M, H], got {tuple(h.shape)}")
    m, hsz = h.shape
    if weights is None:
        places = 1
        if y.shape != (m, hsz) and y.shape != (m, 1, hsz):
            raise ValueError(f"y must be [{m}, {hsz}] without weights, got {tuple(y.shape)}")
    else:
        _check(weights, "weights", (torch.float32,), device)
        places = weights.shape[-1]
        if weights.shape != (m, places) or y.shape != (m, places, hsz):
            raise ValueError(f"weights {tuple(weights.shape)} and y {tuple(y.shape)} do not match h {tuple(h.shape)}")
    if post_norm is not None:
        _check_vector(post_norm, "post_norm", hsz, device)
    if next_norm is not None:
        _check_vector(next_norm, "next_norm", hsz, device)
    row = col = 0
    if gate is not None:
        _check(gate, "gate", (torch.bfloat16,), device)
        strides = {(hsz,): (0, 1), (m, 1): (1, 0), (m, hsz): (hsz, 1)}.get(tuple(gate.shape))
        if strides is None:
            raise ValueError(f"gate must be [{hsz}], [{m}, 1] or [{m}, {hsz}], got {tuple(gate.shape)}")
        row, col = strides
    if out_sq is not None:
        _check(out_sq, "out_sq", (torch.float32,), device)
        if out_sq.numel() < m:
            raise ValueError(f"out_sq needs {m} elements")
    out = _moe_out(out, (m, hsz), h)
    z = h.new_empty((m, hsz)) if next_norm is not None else None
    _lib.call("im_block_residual", y.data_ptr(), _ptr_or_none(weights), places, h.data_ptr(), _ptr_or_none(post_norm),
              _ptr_or_none(gate), row, col, float(residual_scale), _ptr_or_none(next_norm), float(eps), int(gemma), m, hsz,
              out.data_ptr(), _ptr_or_none(z), _ptr_or_none(out_sq), _stream(device))
    return out, z


# ---- decoding over a bounded cache ----------------------------------------------------------------------------
_TYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_LAYOUTS = {"half": _lib.ROPE_HALF, "interleaved": _lib.ROPE_INTERLEAVED}
PAGE_SLOTS = 16


# entry point -> its number in im_bounded_call and its arguments' words: integers and pointers, or one double
_WORDS = {"im_rope": (0, struct.Struct("=9qd10q").pack), "im_rope_kv": (1, struct.Struct("=5qd19q").pack),
          "im_attention_weights": (2, struct.Struct("=21qd7q").pack), "im_cache_evict": (3, struct.Struct("=25q").pack),
          "im_verify_sampled": (4, struct.Struct("=17q").pack)}


def _launch(index: int, name: str, *args) -> None:
    """Call an entry point on a device's current stream (its last argument), with the device current; no tensor is 0."""
    entry, pack = _WORDS[name]
    if torch._C._cuda_getDevice() == index:
        try:
            words = pack(entry, *args, torch._C._cuda_getCurrentRawStream(index))
        except struct.error as exc:
            raise ValueError(f"{name}: an argument is no 64-bit integer ({exc})") from exc
        status = _lib.load().im_bounded_call(words, len(words))
        if status:
            _lib.check(name, status)
    else:
        with torch.cuda.device(index):
            _launch(index, name, *args)


def _ptr_or_zero(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _need(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device, index: int) -> None:
    """_check for one type; what fits costs a third of it."""
    try:
        if t.dtype is dtype and t.get_device() == index and t.is_contiguous():
            return
    except AttributeError:  # no tensor
        pass
    _check(t, name, (dtype,), device)


def _apart(a: torch.Tensor, name_a: str, b: torch.Tensor, name_b: str) -> None:
    """_disjoint_or_same of contiguous tensors of one shape and four-byte type."""
    if 0 < abs(a.data_ptr() - b.data_ptr()) < 4 * a.numel():
        raise ValueError(f"{name_a} overlaps {name_b} without being the same tensor")


def _disjoint_or_same(a: torch.Tensor, name_a: str, b: torch.Tensor, name_b: str) -> None:
    """Refuse tensors that overlap without being one (strides are not negative)."""
    if a is b:
        return

    def end(t: torch.Tensor) -> int:
        if t.is_contiguous():
            return t.data_ptr() + t.numel() * t.element_size()
        last = sum((n - 1) * st for n, st in zip(t.shape, t.stride())) if t.numel() else -1
        return t.data_ptr() + (last + 1) * t.element_size()

    a0, b0 = a.data_ptr(), b.data_ptr()
    if a0 < end(b) and b0 < end(a) and not (a0 == b0 and a.shape == b.shape and a.stride() == b.stride()):
        raise ValueError(f"{name_a} overlaps {name_b} without being the same tensor")


def rope_frequencies(rotary: int, base: float, *, scaling: str = "none", stretch: float = 1.0, trained: int = 0,
                     fast: float = 32.0, slow: float = 1.0,
                     device: torch.device | str = "cuda") -> tuple[torch.Tensor, float]:
    """(inv_freq float64 [rotary / 2], factor) for rope and rope_kv: pair i turns by base^(-2i / rotary) per position.
    scaling for contexts `stretch` times the `trained` length: "linear" (every frequency divided by it), "ntk" (the base
    raised so that the slowest pair's is divided by it), "yarn" (pairs of over `fast` turns over the trained length as they
    are, of under `slow` turns divided, a ramp between; values multiplied by factor = 0.1 ln(stretch) + 1)."""
    if rotary < 2 or rotary % 2:
        raise ValueError(f"rotary {rotary}: an even number of values")
    if not (base > 1.0 and math.isfinite(base)):
        raise ValueError(f"base {base}: a finite number above 1")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"scaling {scaling!r}: none, linear, ntk or yarn")
    if scaling != "none" and not (stretch >= 1.0 and math.isfinite(stretch)):
        raise ValueError(f"stretch {stretch}: at least 1")
    i = torch.arange(rotary // 2, dtype=torch.float64)
    factor = 1.0
    if scaling == "ntk":
        if rotary < 4:
            raise ValueError("ntk scaling needs two pairs or more")
        base = base * stretch ** (rotary / (rotary - 2))
    freq = base ** (-2.0 * i / rotary)
    if scaling == "linear":
        freq = freq / stretch
    elif scaling == "yarn":
        if trained < 1 or not fast > slow > 0.0:
            raise ValueError("yarn scaling needs the trained length, and fast > slow > 0 turns")
        pair = [rotary * math.log(trained / (turns * 2.0 * math.pi)) / (2.0 * math.log(base)) for turns in (fast, slow)]
        low, high = max(0, math.floor(pair[0])), min(rotary - 1, math.ceil(pair[1]))
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        freq = freq / stretch * ramp + freq * (1.0 - ramp)
        factor = 0.1 * math.log(stretch) + 1.0
    return freq.to(device), factor


def _rope_table(inv_freq: torch.Tensor, layout: str, d: int, device: torch.device, index: int) -> tuple[int, int, int]:
    """(rotary, layout, whether in float64) of a table checked against the head size."""
    wide = isinstance(inv_freq, torch.Tensor) and inv_freq.dtype is torch.float64
    _need(inv_freq, "inv_freq", torch.float64 if wide else torch.float32, device, index)
    lay = _LAYOUTS.get(layout)
    if lay is None:
        raise ValueError(f"layout {layout!r}: half or interleaved")
    rotary = 2 * inv_freq.numel()
    if inv_freq.dim() != 1 or rotary > d:
        raise ValueError(f"inv_freq {tuple(inv_freq.shape)} turns {rotary} of a head's {d} values")
    return rotary, lay, int(wide)


def rope(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, layout: str = "half", factor: float = 1.0,
         inverse: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [M, H, D] (bf16, float16 or float32; any row and head strides) turned to positions [M] (int32 or int64): pair i
    of a head's first 2 * len(inv_freq) values by positions * inv_freq[i], times factor; the rest is copied. Pairs are
    (i, i + half of them) or, "interleaved", (2i, 2i + 1). inverse turns back by the transpose: rope(dy, ..., inverse=True)
    is the gradient of x, which autograd does not take by itself. An angle is a float64 product, within 2^-51 of itself.
    `out` may be x; a new tensor by default."""
    kind = _TYPES.get(x.dtype) if isinstance(x, torch.Tensor) and x.is_cuda else None
    if kind is None:
        raise TypeError("x must be a bf16, float16 or float32 CUDA tensor")
    shape, strides = x.shape, x.stride()
    if len(shape) != 3 or (strides[2] != 1 and shape[2] > 1 and x.numel()):
        raise ValueError(f"x must be [M, H, D] with contiguous heads, got {tuple(shape)}, strides {strides}")
    m, h, d = shape
    device = x.device
    index = device.index
    wide = isinstance(positions, torch.Tensor) and positions.dtype is torch.int64
    _need(positions, "positions", torch.int64 if wide else torch.int32, device, index)
    if positions.shape != (m,):
        raise ValueError(f"positions must be [{m}], got {tuple(positions.shape)}")
    rotary, lay, freq64 = _rope_table(inv_freq, layout, d, device, index)
    if out is None:
        out = x.new_empty(m, h, d)
        rs, hs = h * d, d
    else:
        if not isinstance(out, torch.Tensor) or out.dtype != x.dtype or out.device != device or out.shape != shape:
            raise ValueError(f"out must be a {x.dtype} tensor {tuple(shape)} on {device}")
        rs, hs, by_value = out.stride()
        by_row = (h < 2 or hs >= d) and (m < 2 or rs >= (h - 1) * hs + d)
        by_head = (m < 2 or rs >= d) and (h < 2 or hs >= (m - 1) * rs + d)
        if out.numel() and ((d > 1 and by_value != 1) or not (by_row or by_head)):
            raise ValueError(f"out must hold every head apart and contiguous, its strides are {out.stride()}")
        _disjoint_or_same(out, "out", x, "x")
    if m and h and d:
        _launch(index, "im_rope", x.data_ptr(), strides[0], strides[1], positions.data_ptr(), int(wide),
                inv_freq.data_ptr(), freq64, rotary, float(factor), lay, int(inverse), m, h, d, kind, out.data_ptr(), rs, hs)
    return out


def _check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, hkv: int, d: int, dtype,
                 device: torch.device, index: int) -> tuple[int, int, int]:
    """(sequences, pages a sequence, pages) of caches [pages, Hkv, 16, D] and their page table."""
    _need(k_cache, "k_cache", dtype, device, index)
    _need(v_cache, "v_cache", dtype, device, index)
    shape = k_cache.shape
    if v_cache.shape != shape or len(shape) != 4 or shape[1:] != (hkv, PAGE_SLOTS, d):
        raise ValueError(f"caches must be [pages, {hkv}, {PAGE_SLOTS}, {d}], got {tuple(k_cache.shape)} and "
                         f"{tuple(v_cache.shape)}")
    _need(page_table, "page_table", torch.int32, device, index)
    table = page_table.shape
    if len(table) != 2:
        raise ValueError(f"page_table must be [sequences, pages], got {tuple(page_table.shape)}")
    return table[0], table[1], shape[0]


def _check_ints(t: torch.Tensor, name: str, n: int, device: torch.device, index: int) -> None:
    _need(t, name, torch.int32, device, index)
    if t.dim() != 1 or t.numel() < n:
        raise ValueError(f"{name} must hold {n} elements, got {tuple(t.shape)}")


def _check_slots(t: torch.Tensor, name: str, dtype, lead: tuple, device: torch.device, index: int) -> int:
    """cap of a [..., sequences, Hkv, cap] tensor; lead: all but cap."""
    _need(t, name, dtype, device, index)
    shape = t.shape
    if len(shape) != len(lead) + 1 or shape[:-1] != lead:
        raise ValueError(f"{name} must be [{', '.join(map(str, lead))}, slots], got {tuple(t.shape)}")
    return shape[-1]


def rope_kv(qkv: torch.Tensor, inv_freq: torch.Tensor, row_pos: torch.Tensor, row_slot: torch.Tensor,
            row_seq: torch.Tensor, page_table: torch.Tensor, hq: int, hkv: int, d: int, k_cache: torch.Tensor,
            v_cache: torch.Tensor, *, layout: str = "half", factor: float = 1.0, q_out: torch.Tensor | None = None,
            slot_pos: torch.Tensor | None = None, rows: int | None = None) -> torch.Tensor:
    """The first `rows` rows of qkv [M, (Hq + 2 Hkv) D] (bf16, float16 or float32): q turned to its position (returned,
    [M, Hq, D]), k turned and v written to slot row_slot of table row row_seq of the caches [pages, Hkv, 16, D], and, with
    slot_pos (int32 [sequences, Hkv, cap]), the position to that slot of every head. Rows whose slot is outside the table
    (-1) write no cache; no two rows may name one slot. What rope says of inv_freq, layout and factor holds."""
    if not (isinstance(qkv, torch.Tensor) and qkv.is_cuda and qkv.dtype in _TYPES and qkv.is_contiguous()):
        _check(qkv, "qkv", _FLOATS)
    device, dtype = qkv.device, qkv.dtype
    index = device.index
    if hq < 1 or hkv < 1 or hq % hkv or d < 1:
        raise ValueError(f"{hq} query heads, {hkv} kv heads of {d} values")
    if qkv.dim() != 2 or qkv.shape[1] != (hq + 2 * hkv) * d:
        raise ValueError(f"qkv must be [M, {(hq + 2 * hkv) * d}], got {tuple(qkv.shape)}")
    m = qkv.shape[0] if rows is None else rows
    if not 0 <= m <= qkv.shape[0]:
        raise ValueError(f"{m} rows of {qkv.shape[0]}")
    rotary, lay, freq64 = _rope_table(inv_freq, layout, d, device, index)
    for t, name in ((row_pos, "row_pos"), (row_slot, "row_slot"), (row_seq, "row_seq")):
        _check_ints(t, name, m, device, index)
    seqs, max_pages, pages = _check_cache(k_cache, v_cache, page_table, hkv, d, dtype, device, index)
    cap = 0 if slot_pos is None else _check_slots(slot_pos, "slot_pos", torch.int32, (seqs, hkv), device, index)
    if q_out is None:
        q_out = qkv.new_empty(m, hq, d)
    else:
        _need(q_out, "q_out", dtype, device, index)
        if q_out.numel() < m * hq * d:
            raise ValueError(f"q_out needs {m * hq * d} elements")
        _disjoint_or_same(q_out, "q_out", qkv, "qkv")
        if q_out.data_ptr() == qkv.data_ptr():
            raise ValueError("q_out must not be qkv")
    if m:
        _launch(index, "im_rope_kv", qkv.data_ptr(), inv_freq.data_ptr(), freq64, rotary, float(factor), lay,
                row_pos.data_ptr(), row_slot.data_ptr(), row_seq.data_ptr(), page_table.data_ptr(), seqs, max_pages, pages,
                m, hq, hkv, d, _TYPES[dtype],
                q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _ptr_or_zero(slot_pos), cap)
    return q_out


@functools.lru_cache(maxsize=4096)
def _attention_weights_workspace(b: int, rows: int, hq: int, hkv: int, d: int, kv: int, kps: int, window: int) -> int:
    return int(_lib.load().im_attention_weights_workspace_bytes(b, rows, hq, hkv, d, kv, kps, window))


def attention_weights(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                      seq_rows: torch.Tensor, row_slot: torch.Tensor, weights: torch.Tensor, *, max_rows_per_seq: int,
                      max_kv_len: int, scale: float, keys_per_split: int = 0, window: int = 0,
                      weights_out: torch.Tensor | None = None, out: torch.Tensor | None = None, rows: int | None = None,
                      seq_slot: torch.Tensor | None = None) -> torch.Tensor:
    """Paged attention of new rows, q [M, Hq, D] -> out [M, Hq, D] (bf16 or float16, D a multiple of 16 up to 256), that
    adds up each slot's attention weight: weights (float32 [sequences, Hkv, cap], the rows of the page table) becomes, in
    place or in weights_out, weights + the softmax weights that the sequence's rows and the kv head's query heads put on
    the slot, for the slots up to the last row's; from the slot of the first row that has one on it starts from zero. Rows
    without a slot (-1) get zeros and add nothing. `out` may be q. No two sequences may name one table row. The other arguments
    are `attention`'s, keys_per_split 0 meaning that the call's sizes choose it, for the least time of a call from Python: in a
    captured graph a length that makes more than 16 splits can be faster (one row of 32/8 heads over 5000 slots 11.6 us
    with two kernels, 13.7 with the one that is chosen)."""
    dtype = torch.float16 if isinstance(q, torch.Tensor) and q.dtype is torch.float16 else torch.bfloat16
    if not (isinstance(q, torch.Tensor) and q.is_cuda and q.dtype is dtype and q.is_contiguous()):
        _check(q, "q", (torch.bfloat16, torch.float16))
    device = q.device
    index = device.index
    if q.dim() != 3 or not isinstance(k_cache, torch.Tensor) or k_cache.dim() != 4:
        raise ValueError(f"q must be [M, Hq, D] and the caches [pages, Hkv, 16, D], got q {tuple(q.shape)}")
    held, hq, d = q.shape
    hkv = k_cache.shape[1]
    m = held if rows is None else rows
    if not 0 <= m <= held:
        raise ValueError(f"{m} rows of {held}")
    if hkv < 1 or hq < 1 or hq % hkv:
        raise ValueError(f"{hq} query heads, {hkv} kv heads")
    seqs, max_pages, pages = _check_cache(k_cache, v_cache, page_table, hkv, d, dtype, device, index)
    _check_ints(seq_rows, "seq_rows", 1, device, index)
    b = seq_rows.numel() - 1
    _check_ints(row_slot, "row_slot", m, device, index)
    if seq_slot is not None:
        _check_ints(seq_slot, "seq_slot", b, device, index)
    elif b > seqs:
        raise ValueError(f"{b} sequences, the page table has {seqs}")
    cap = _check_slots(weights, "weights", torch.float32, (seqs, hkv), device, index)
    if weights_out is None:
        weights_out = weights
    else:
        _need(weights_out, "weights_out", torch.float32, device, index)
        if weights_out.shape != weights.shape:
            raise ValueError(f"weights_out must be {tuple(weights.shape)}, got {tuple(weights_out.shape)}")
        _apart(weights_out, "weights_out", weights, "weights")
    if out is None:
        out = q.new_empty(m, hq, d)  # sizes one by one: 0.4 us less than a tuple of them
    else:
        _need(out, "out", dtype, device, index)
        if out.numel() < m * hq * d:
            raise ValueError(f"out needs {m * hq * d} elements")
        _disjoint_or_same(out, "out", q, "q")
    if not (0 <= max_rows_per_seq and 0 <= max_kv_len and 0 <= window and 0 <= keys_per_split):
        raise ValueError("max_rows_per_seq, max_kv_len, window and keys_per_split are not negative")
    if b == 0 or m == 0 or max_rows_per_seq == 0:
        return out
    max_rows = min(max_rows_per_seq, m)
    need = _attention_weights_workspace(b, max_rows, hq, hkv, d, max(1, max_kv_len), keys_per_split, window)
    ws = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=device) if need else None  # few, short splits need none
    _launch(index, "im_attention_weights", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _TYPES[dtype],
            page_table.data_ptr(), seqs, max_pages, pages, seq_rows.data_ptr(),
            _ptr_or_zero(seq_slot), row_slot.data_ptr(), m, b, max_rows, hq, hkv, d, max_kv_len, keys_per_split, window,
            float(scale), weights.data_ptr(), weights_out.data_ptr(), cap, out.data_ptr(), _ptr_or_zero(ws),
            need)
    return out


@functools.lru_cache(maxsize=4096)
def _evict_workspace(layers: int, s: int, hkv: int, cap: int, budget: int) -> int:
    return int(_lib.load().im_cache_evict_workspace_bytes(layers, s, hkv, cap, budget))


def cache_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                seen: torch.Tensor, weights: torch.Tensor, slot_pos: torch.Tensor, *, budget: int, recent: int = 0,
                sinks: int = 0, weights_out: torch.Tensor | None = None, pos_out: torch.Tensor | None = None,
                lengths_out: torch.Tensor | None = None) -> torch.Tensor:
    """Cut every kv head's slots to `budget`, in place, and return the new lengths (int32 [sequences]). Of the lengths[s]
    slots of a head, those stay that hold a token below position `sinks` or among the last `recent` of the seen[s] tokens of
    the sequence, and the ones with the largest weights (lower slots first among equals); kept slots behind the new end
    move into the holes before it. weights (float32) and slot_pos (int32) are [sequences, Hkv, cap] and follow, in place
    or to weights_out and pos_out. Caches [pages, Hkv, 16, D] of any type, or [layers, pages, Hkv, 16, D] with weights
    and slot_pos [layers, sequences, Hkv, cap]: every layer of one call makes its own choice. Page tables must not share the
    pages that are cut."""
    if not isinstance(k_cache, torch.Tensor) or k_cache.dim() not in (4, 5):
        raise ValueError("caches must be [pages, Hkv, 16, D] or [layers, pages, Hkv, 16, D]")
    device, dtype = k_cache.device, k_cache.dtype
    index = device.index
    if not (k_cache.is_cuda and k_cache.is_contiguous()):
        _check(k_cache, "k_cache", (dtype,))
    _need(v_cache, "v_cache", dtype, device, index)
    if v_cache.shape != k_cache.shape or k_cache.shape[-2] != PAGE_SLOTS:
        raise ValueError(f"caches must be of one shape with {PAGE_SLOTS} slots a page, got {tuple(k_cache.shape)} and "
                         f"{tuple(v_cache.shape)}")
    shape = k_cache.shape
    layers = shape[0] if len(shape) == 5 else 1
    pages, hkv, _, d = shape[-4:]
    _need(page_table, "page_table", torch.int32, device, index)
    if page_table.dim() != 2:
        raise ValueError(f"page_table must be [sequences, pages], got {tuple(page_table.shape)}")
    s, max_pages = page_table.shape
    for t, name in ((lengths, "lengths"), (seen, "seen"), (lengths_out, "lengths_out")):
        if t is not None or name != "lengths_out":
            _need(t, name, torch.int32, device, index)
            if t.shape != (s,):
                raise ValueError(f"{name} must be [{s}], got {tuple(t.shape)}")
    lead = (layers, s, hkv) if len(shape) == 5 else (s, hkv)
    cap = _check_slots(weights, "weights", torch.float32, lead, device, index)
    if _check_slots(slot_pos, "slot_pos", torch.int32, lead, device, index) != cap:
        raise ValueError(f"slot_pos is {tuple(slot_pos.shape)}, weights {tuple(weights.shape)}")
    for t, name, like, like_name in ((weights_out, "weights_out", weights, "weights"),
                                     (pos_out, "pos_out", slot_pos, "slot_pos")):
        if t is not None:
            _need(t, name, like.dtype, device, index)
            if t.shape != like.shape:
                raise ValueError(f"{name} must be {tuple(like.shape)}, got {tuple(t.shape)}")
            _apart(t, name, like, like_name)
    if lengths_out is None:
        lengths_out = torch.empty_like(lengths)
    else:
        _apart(lengths_out, "lengths_out", lengths, "lengths")
        if s and lengths_out.data_ptr() < seen.data_ptr() + 4 * s and seen.data_ptr() < lengths_out.data_ptr() + 4 * s:
            raise ValueError("lengths_out overlaps seen")
    if budget < 0 or recent < 0 or sinks < 0 or recent + sinks > budget:
        raise ValueError(f"{recent} recent and {sinks} first slots of a budget of {budget}")
    if not (layers and s and hkv and cap and d):
        return lengths_out.zero_()
    need = _evict_workspace(layers, s, hkv, cap, budget)
    ws = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=device) if need else None  # few moves a row need none
    size = k_cache.element_size()
    _launch(index, "im_cache_evict", k_cache.data_ptr(), v_cache.data_ptr(), layers, pages * hkv * PAGE_SLOTS * d * size,
            pages, page_table.data_ptr(), max_pages, lengths.data_ptr(), seen.data_ptr(), weights.data_ptr(),
            (weights if weights_out is None else weights_out).data_ptr(), slot_pos.data_ptr(),
            (slot_pos if pos_out is None else pos_out).data_ptr(), lengths_out.data_ptr(), s, hkv, cap, d * size,
            budget, recent, sinks, _ptr_or_zero(ws), need)
    return lengths_out


def _check_probs(t: torch.Tensor, name: str, rows: int, index: int | None) -> int:
    """The row stride of probabilities [B, rows, V] whose rows are evenly spaced."""
    if not t.is_cuda or t.dtype not in _TYPES:
        raise TypeError(f"{name} must be a bf16, float16 or float32 CUDA tensor")
    if index is not None and t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")
    b, _, v = t.shape
    if t.is_contiguous():
        return v
    by_b, by_row, by_v = t.stride()
    ld = by_row if rows > 1 else by_b if b > 1 else v
    if (v > 1 and by_v != 1) or ld < v or (b > 1 and by_b != rows * ld):
        raise ValueError(f"{name} must have evenly spaced rows of contiguous values, its strides are {t.stride()}")
    return ld


def _check_verified(tokens: torch.Tensor | None, count: torch.Tensor | None, drafts: torch.Tensor, uniforms: torch.Tensor,
                    n_drafts: torch.Tensor | None) -> None:
    """Refuse outputs that lie over inputs of another sequence, which may still be read. A sequence's own are read by then,
    but for drafts, which are copied upwards."""
    if tokens is not None and count is not None:
        _disjoint_or_same(tokens, "tokens", count, "count")
    for out, name in ((tokens, "tokens"), (count, "count")):
        if out is None:
            continue
        for t, what in ((drafts, "drafts"), (uniforms, "uniforms"), (n_drafts, "n_drafts")):
            if t is not None and (drafts.shape[0] > 1 or (t is drafts and out.data_ptr() > t.data_ptr())):
                _disjoint_or_same(out, name, t, what)


def verify_sampled(target_probs: torch.Tensor, draft_probs: torch.Tensor | None, drafts: torch.Tensor,
                   uniforms: torch.Tensor, *, n_drafts: torch.Tensor | None = None, tokens: torch.Tensor | None = None,
                   count: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Speculative sampling from probabilities and given random numbers: target_probs [B, k+1, V] and draft_probs
    [B, k, V] (bf16, float16 or float32), drafts int32 [B, k], uniforms float32 [B, k+1] in [0, 1) -> (tokens int32
    [B, k+1]: the kept drafts, the drawn token, then -1; count int32 [B]). Draft i is kept iff those before it are and
    u[i] * q(d) < p(d); the token after them is drawn with u[k] from max(p - q, 0), or from p after the last draft.
    draft_probs None: drafts without a distribution (n-gram drafts), kept iff u[i] < p(d), else drawn from p without d.
    n_drafts int32 [B]: sequences with fewer drafts than k."""
    if not isinstance(drafts, torch.Tensor) or drafts.dim() != 2:
        raise ValueError("drafts must be [B, k]")
    b, k = drafts.shape
    if not isinstance(target_probs, torch.Tensor) or target_probs.dim() != 3 or target_probs.shape[:2] != (b, k + 1):
        raise ValueError(f"target_probs must be [{b}, {k + 1}, V]")
    v = target_probs.shape[2]
    if v < 1:
        raise ValueError("target_probs has an empty vocabulary")
    p_ld = _check_probs(target_probs, "target_probs", k + 1, None)
    device = target_probs.device
    index = device.index
    q_ld = 0
    if draft_probs is not None:
        if not isinstance(draft_probs, torch.Tensor) or draft_probs.shape != (b, k, v):
            raise ValueError(f"draft_probs must be [{b}, {k}, {v}]")
        if draft_probs.dtype != target_probs.dtype:
            raise TypeError(f"draft_probs is {draft_probs.dtype}, target_probs {target_probs.dtype}")
        q_ld = _check_probs(draft_probs, "draft_probs", k, index) if k else v
    _need(drafts, "drafts", torch.int32, device, index)
    _need(uniforms, "uniforms", torch.float32, device, index)
    if uniforms.shape != (b, k + 1):
        raise ValueError(f"uniforms must be [{b}, {k + 1}], got {tuple(uniforms.shape)}")
    for t, name, shape in ((n_drafts, "n_drafts", (b,)), (tokens, "tokens", (b, k + 1)), (count, "count", (b,))):
        if t is not None:
            _need(t, name, torch.int32, device, index)
            if t.shape != shape:
                raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    if tokens is not None or count is not None:
        _check_verified(tokens, count, drafts, uniforms, n_drafts)
    tokens = drafts.new_empty(b, k + 1) if tokens is None else tokens
    count = drafts.new_empty(b) if count is None else count
    if b:
        _launch(index, "im_verify_sampled", target_probs.data_ptr(), p_ld, _ptr_or_zero(draft_probs), q_ld,
                _TYPES[target_probs.dtype], drafts.data_ptr(), k, _ptr_or_zero(n_drafts), uniforms.data_ptr(), k + 1, b, k,
                v, tokens.data_ptr(), count.data_ptr())
    return tokens, count


# ---- GGUF k-quants (the ggml path) ----------------------------------------------------------------------------
Q4_K, Q6_K = 12, 14
KQ_BLOCK_BYTES = {Q4_K: 144, Q6_K: 210}


def kq_workspace_bytes(k: int, b: int) -> int:
    return int(_lib.load().im_kq_workspace_bytes(k, b))


def _kq_args(kind: int, w: torch.Tensor, x: torch.Tensor, n: int, out: torch.Tensor | None):
    if kind not in KQ_BLOCK_BYTES:
        raise ValueError(f"weight type {kind}: 12 (Q4_K) or 14 (Q6_K)")
    _check(w, "w", (torch.uint8,))
    _check(x, "x", (torch.float32,), w.device)
    if x.dim() != 2:
        raise ValueError("x must be [B, K]")
    b, k = x.shape
    if k % 256 or w.numel() != n * (k // 256) * KQ_BLOCK_BYTES[kind]:
        raise ValueError(f"w holds {w.numel()} bytes, expected {n} rows of {k // 256} blocks")
    y = torch.empty((b, n), dtype=torch.float32, device=w.device) if out is None else out
    _check(y, "out", (torch.float32,), w.device)
    if tuple(y.shape) != (b, n):
        raise ValueError(f"out must be [{b}, {n}]")
    return b, k, y


def kq_gemv(kind: int, w: torch.Tensor, x: torch.Tensor, n: int, *, out: torch.Tensor | None = None,
            ws: torch.Tensor | None = None) -> torch.Tensor:
    """y [B, N] float32 = x [B, K] float32 . W^T, W = N rows of GGUF Q4_K / Q6_K blocks as raw bytes (uint8)."""
    b, k, y = _kq_args(kind, w, x, n, out)
    ws_ptr, ws_bytes = _scratch(ws, w.device, kq_workspace_bytes(k, b), "kq")
    _lib.call("im_kq_gemv", kind, w.data_ptr(), x.data_ptr(), y.data_ptr(), n, k, b, ws_ptr, ws_bytes,
              _stream(w.device))
    return y


def kq_mul_mat(kind: int, w: torch.Tensor, x: torch.Tensor, n: int, *,
               out: torch.Tensor | None = None) -> tuple[int, torch.Tensor]:
    """The llama.cpp hook's call (`ironmule_kg_mul_mat`): (0, y) when y was computed, else (the library's refusal
    code, y unwritten) and the caller runs its own kernel."""
    b, k, y = _kq_args(kind, w, x, n, out)
    rc = int(_lib.load().im_kq_mul_mat(kind, w.data_ptr(), x.data_ptr(), y.data_ptr(), n, k, b,
                                       _stream(w.device)))
    return rc, y
