"""Attention over a paged K/V cache: many sequences in one pool of pages.

``kv_write`` / ``decode`` / ``prefill`` (attention.py) take one contiguous cache per sequence, as
the reference's runners hold one (gemma4_150/runner.py:344-441). A server that holds many
sequences of unknown length keeps their rows in pages instead:

  * ``k_pages`` / ``v_pages`` [n_pages][page_size][kvH][hd], f16 or f32, page_size a power of two
    from 16;
  * ``page_table`` int32 [n_seq][cols]: position p of sequence b is row p % page_size of page
    ``page_table[b][p // page_size]``. An entry outside [0, n_pages) is a page that is not there:
    its positions are neither written nor attended (-1 for pages behind a sliding window);
  * ``key_len`` int32 [n_seq]: the keys of each sequence, this call's tokens included; 0 = idle;
  * ``cu_q`` int32 [n_seq + 1]: packed rows cu_q[b] .. cu_q[b+1]-1 are sequence b's tokens, its last
    ones. Rows from cu_q[n_seq] on belong to nobody: not read, their outputs left as they were;
  * ``rope_cos`` / ``rope_sin`` f32 [>= max_key_len][hd/2]: ``rope_tables`` over absolute positions.

All of these live on one GPU, so lengths and tables can change between replays of a captured
graph. ``max_key_len`` is the host's bound of key_len (default: all that the table's columns
hold); it sizes grids and workspaces, and a longer key_len is taken as max_key_len.

A step of such a server, per layer: ``paged_write`` the prompts' k/v rows, then ``paged_prefill``
their queries; then one ``paged_decode`` per generated token, which appends the token's own row.
Calls run on the current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import G4APaged, check
from .attention import AttnConfig, DecodeWorkspace, _need, _ptr

__all__ = ["paged_write", "paged_decode", "paged_decode_ws_bytes", "paged_prefill", "paged_prefill_ws_bytes"]

_F32, _F16, _I32 = torch.float32, torch.float16, torch.int32


def _same_device(dev, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the other operands on {dev}")


def _on_device(dev, fn, *args):
    """fn(*args, stream) with dev current: the kernels launch on the current device."""
    if dev.index == torch.cuda.current_device():
        return fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    with torch.cuda.device(dev):
        return fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))


def _cache(dev, k_pages, v_pages, page_table, key_len, cfg, max_key_len, rope_cos, rope_sin) -> G4APaged:
    """The checked g4a_paged of a call."""
    if k_pages.dim() != 4 or k_pages.shape[2:] != (cfg.n_kv_heads, cfg.head_dim) or v_pages.shape != k_pages.shape:
        raise ValueError(f"k_pages / v_pages must be [n_pages][page_size][{cfg.n_kv_heads}][{cfg.head_dim}], got "
                         f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    if k_pages.dtype != v_pages.dtype or k_pages.dtype not in (_F16, _F32):
        raise ValueError("k/v pages must both be float16 or both float32")
    _need(k_pages, "k_pages")
    _need(v_pages, "v_pages")
    if not page_table.is_cuda or page_table.dtype is not _I32 or page_table.dim() != 2 or page_table.stride(1) != 1:
        raise ValueError("page_table must be an int32 device tensor [n_seq][cols] with adjacent columns")
    n_seq, cols = page_table.shape
    stride = page_table.stride(0) if n_seq > 1 else cols
    if stride < cols:
        raise ValueError("page_table rows must not overlap")
    _need(key_len, "key_len", _I32)
    if key_len.numel() != n_seq:
        raise ValueError(f"key_len must have one entry per row of page_table ({n_seq}), got {key_len.numel()}")
    page = k_pages.shape[1]
    if max_key_len is None:
        max_key_len = cols * page
        if rope_cos is not None:
            max_key_len = min(max_key_len, rope_cos.shape[0])
    if not 0 < max_key_len <= cols * page:
        raise ValueError(f"max_key_len must be in [1, {cols * page}], what the page table's columns hold")
    if (rope_cos is None) != (rope_sin is None):
        raise ValueError("rope_cos and rope_sin go together")
    if rope_cos is not None:
        _need(rope_cos, "rope_cos", _F32)
        _need(rope_sin, "rope_sin", _F32)
        if rope_cos.dim() != 2 or rope_cos.shape[1] != cfg.head_dim // 2 or rope_cos.shape[0] < max_key_len or (
                rope_sin.shape != rope_cos.shape):
            raise ValueError(f"rope tables must be [>= max_key_len ({max_key_len})][head_dim/2], got "
                             f"{tuple(rope_cos.shape)} and {tuple(rope_sin.shape)}")
    _same_device(dev, k_pages=k_pages, v_pages=v_pages, page_table=page_table, key_len=key_len, rope_cos=rope_cos,
                 rope_sin=rope_sin)
    return G4APaged(k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), key_len.data_ptr(), k_pages.shape[0],
                    page, n_seq, cols, stride, int(max_key_len))


def _cu(cu_q, n_seq, dev):
    _need(cu_q, "cu_q", _I32)
    if cu_q.numel() != n_seq + 1:
        raise ValueError(f"cu_q must have n_seq + 1 = {n_seq + 1} entries, got {cu_q.numel()}")
    _same_device(dev, cu_q=cu_q)


def paged_write(k, v, k_pages, v_pages, page_table, key_len, cu_q, cfg: AttnConfig, *, k_gain=None, rope_cos=None,
                rope_sin=None, k_in_q: float = 0.0, v_in_q: float = 0.0, v_norm: bool = True,
                max_key_len: int | None = None):
    """Append packed tokens' k/v rows ([T][kvH][hd], f32 or f16) to the cache.

    Each row is prepared as ``kv_write`` prepares it, to the bit: srq with k_in_q / v_in_q,
    k RMSNorm * k_gain and RoPE at its position, v RMSNorm."""
    if k.dim() != 3 or k.shape[1:] != (cfg.n_kv_heads, cfg.head_dim) or v.shape != k.shape or k.dtype != v.dtype:
        raise ValueError(f"k/v shape {tuple(k.shape)} does not match {cfg}")
    _need(k, "k", (_F16, _F32))
    _need(v, "v", (_F16, _F32))
    _need(k_gain, "k_gain", _F32)
    dev = k.device
    pg = _cache(dev, k_pages, v_pages, page_table, key_len, cfg, max_key_len, rope_cos, rope_sin)
    _cu(cu_q, pg.n_seq, dev)
    _same_device(dev, v=v, k_gain=k_gain)
    c = cfg.c((_lib.KV_F32 if k_pages.dtype is _F32 else 0) | (_lib.IN_F16 if k.dtype is _F16 else 0) |
              (0 if v_norm else _lib.NO_V_NORM))
    check(_on_device(dev, _lib.load().g4a_paged_write, ctypes.byref(c), ctypes.byref(pg), k.shape[0], _ptr(cu_q), _ptr(k),
                     _ptr(v), float(k_in_q), float(v_in_q), _ptr(k_gain), _ptr(rope_cos), _ptr(rope_sin)))


def _out(out, q, out_dtype):
    if out is None:
        return torch.empty(q.shape, dtype=out_dtype, device=q.device)
    if out.shape != q.shape:
        raise ValueError(f"out must be shaped like q {tuple(q.shape)}, got {tuple(out.shape)}")
    return out


def _q(q, cfg, q_gain):
    if q.dim() != 3 or q.shape[1:] != (cfg.n_q_heads, cfg.head_dim):
        raise ValueError(f"q shape {tuple(q.shape)} does not match {cfg}")
    _need(q, "q", _F32)
    _need(q_gain, "q_gain", _F32)


def _sizes(n_pages, page_size, n_seq, cols, max_key_len) -> G4APaged:
    # a size needs no memory: addresses that pass the checks and are never followed
    return G4APaged(256, 256, 256, 256, n_pages, page_size, n_seq, cols, cols, max_key_len)


def paged_decode_ws_bytes(n_seq: int, max_key_len: int, cfg: AttnConfig, *, page_size: int, kv_f32: bool = False) -> int:
    """Workspace bytes of a ``paged_decode`` call (g4a_paged_decode_ws_bytes): reserve the largest call's."""
    c = cfg.c(_lib.KV_F32 if kv_f32 else 0)
    pg = _sizes(1, page_size, n_seq, -(-max_key_len // page_size), max_key_len)
    n = _lib.load().g4a_paged_decode_ws_bytes(ctypes.byref(c), ctypes.byref(pg))
    if n == 0:
        check(-1)
    return int(n)


def paged_decode(q, k_pages, v_pages, page_table, key_len, cfg: AttnConfig, *, workspace: DecodeWorkspace | None = None,
                 q_gain=None, rope_cos=None, rope_sin=None, k_new=None, v_new=None, k_gain=None, k_in_q: float = 0.0,
                 v_in_q: float = 0.0, v_norm: bool = True, out=None, out_dtype=torch.float16,
                 max_key_len: int | None = None):
    """Attention of one new token per sequence, at position key_len - 1.

    q f32 [n_seq][nH][hd] raw. With k_new / v_new (f32 [n_seq][kvH][hd]) the step's rows are
    prepared as ``kv_write`` prepares them and appended at position key_len - 1 by the same call
    before they are attended. Returns out [n_seq][nH][hd] (f16 by default); an idle sequence's
    rows are zeros. `workspace`: the caller's scratch (paged_decode_ws_bytes)."""
    _q(q, cfg, q_gain)
    dev = q.device
    pg = _cache(dev, k_pages, v_pages, page_table, key_len, cfg, max_key_len, rope_cos, rope_sin)
    if q.shape[0] != pg.n_seq:
        raise ValueError(f"q holds {q.shape[0]} tokens, page_table {pg.n_seq} sequences")
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new go together")
    for name, x in (("k_new", k_new), ("v_new", v_new)):
        _need(x, name, _F32)
        if x is not None and x.shape != (pg.n_seq, cfg.n_kv_heads, cfg.head_dim):
            raise ValueError(f"{name} must be [{pg.n_seq}][{cfg.n_kv_heads}][{cfg.head_dim}]")
    _need(k_gain, "k_gain", _F32)
    out = _out(out, q, out_dtype)
    _need(out, "out", (_F16, _F32))
    _same_device(dev, q_gain=q_gain, k_new=k_new, v_new=v_new, k_gain=k_gain, out=out)
    c = cfg.c((_lib.KV_F32 if k_pages.dtype is _F32 else 0) | (_lib.OUT_F32 if out.dtype is _F32 else 0) |
              (0 if v_norm else _lib.NO_V_NORM))
    lib = _lib.load()
    ws_bytes = lib.g4a_paged_decode_ws_bytes(ctypes.byref(c), ctypes.byref(pg))
    if ws_bytes == 0:
        check(-1)
    ws = (workspace or DecodeWorkspace(dev)).get(ws_bytes)
    _same_device(dev, workspace=ws)
    check(_on_device(dev, lib.g4a_paged_decode, ctypes.byref(c), ctypes.byref(pg), _ptr(q), _ptr(q_gain), _ptr(rope_cos),
                     _ptr(rope_sin), _ptr(k_new), _ptr(v_new), float(k_in_q), float(v_in_q), _ptr(k_gain), _ptr(out),
                     _ptr(ws), ws_bytes))
    return out


def paged_prefill_ws_bytes(n_tokens: int, n_seq: int, max_key_len: int, cfg: AttnConfig, *, page_size: int,
                           kv_f32: bool = False) -> int:
    """Workspace bytes of a ``paged_prefill`` call (g4a_paged_prefill_ws_bytes): reserve the largest call's."""
    c = cfg.c(_lib.KV_F32 if kv_f32 else 0)
    pg = _sizes(1, page_size, n_seq, -(-max_key_len // page_size), max_key_len)
    n = _lib.load().g4a_paged_prefill_ws_bytes(ctypes.byref(c), ctypes.byref(pg), int(n_tokens))
    if n == 0:
        check(-1)
    return int(n)


def paged_prefill(q, k_pages, v_pages, page_table, key_len, cu_q, cfg: AttnConfig, *, workspace: DecodeWorkspace,
                  q_gain=None, rope_cos=None, rope_sin=None, out=None, out_dtype=torch.float16,
                  max_key_len: int | None = None):
    """Causal attention of packed prompts, or pieces of them, whose rows the cache already holds.

    q f32 [T][nH][hd] raw; the normalised, rotated q is rounded to f16 (as ``prefill`` without
    q_hilo). Returns out [T][nH][hd] (f16 by default). f32 caches are converted to f16 in the
    workspace. `workspace`: the caller's scratch (paged_prefill_ws_bytes)."""
    _q(q, cfg, q_gain)
    dev = q.device
    pg = _cache(dev, k_pages, v_pages, page_table, key_len, cfg, max_key_len, rope_cos, rope_sin)
    _cu(cu_q, pg.n_seq, dev)
    out = _out(out, q, out_dtype)
    _need(out, "out", (_F16, _F32))
    _same_device(dev, q_gain=q_gain, out=out)
    c = cfg.c((_lib.KV_F32 if k_pages.dtype is _F32 else 0) | (_lib.OUT_F32 if out.dtype is _F32 else 0))
    lib = _lib.load()
    ws_bytes = lib.g4a_paged_prefill_ws_bytes(ctypes.byref(c), ctypes.byref(pg), q.shape[0])
    if ws_bytes == 0:
        check(-1)
    ws = workspace.get(ws_bytes)
    _same_device(dev, workspace=ws)
    check(_on_device(dev, lib.g4a_paged_prefill, ctypes.byref(c), ctypes.byref(pg), q.shape[0], _ptr(cu_q), _ptr(q),
                     _ptr(q_gain), _ptr(rope_cos), _ptr(rope_sin), _ptr(out), _ptr(ws), ws_bytes))
    return out
