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
    ones. Rows from cu_q[n_seq] on belong to nobody: nothing is stored for them, their outputs stay. A call
    of no packed rows, or no sequences, has nothing to do (its operands are checked all the same);
  * ``rope_cos`` / ``rope_sin`` f32 [>= max_key_len][hd/2]: ``rope_tables`` over absolute positions.

All of these live on one GPU, so lengths and tables can change between replays of a captured
graph. ``max_key_len`` is the host's bound of key_len (default: all that the table's columns and
the RoPE tables hold); it sizes grids and workspaces, and a longer key_len is taken as max_key_len.

A step of such a server, per layer: ``paged_write`` the prompts' k/v rows, then ``paged_prefill``
their queries; then one ``paged_decode`` per generated token, which appends the token's own row.
Calls run on the current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import G4APaged, check
from .attention import AttnConfig, DecodeWorkspace

__all__ = ["paged_write", "paged_decode", "paged_decode_ws_bytes", "paged_prefill", "paged_prefill_ws_bytes"]

_F32, _F16, _I32 = torch.float32, torch.float16, torch.int32
_HALF_OR_FLOAT = (_F16, _F32)
_EWORKSPACE, _I32_MAX = -3, 2 ** 31 - 1


# A decode step of short sequences is bound by this layer, not by its kernels: the checks below touch each
# tensor a few times, whole numbers go to ctypes as they are, and the workspace's size is only asked for
# when the library finds it too small (one sequence of 300 keys 19.2 -> 15 us a call).
def _refuse(name, t, dev, dtype):
    """What is wrong with a tensor that _t found unfit."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, the other operands on cuda:{dev}")
    if t.dtype is not dtype and not (isinstance(dtype, tuple) and t.dtype in dtype):
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    raise ValueError(f"{name} must be contiguous")


def _t(name, t, dev, dtype):
    """Address of a contiguous tensor of dtype on GPU dev; None stays None."""
    if t is None:
        return None
    if t.get_device() != dev or t.dtype is not dtype or not t.is_contiguous():
        _refuse(name, t, dev, dtype)
    return t.data_ptr()


def _gain(name, t, dev, cfg):
    """Address of a norm's gains, one per dim: the kernels read head_dim of them."""
    if t is None:
        return None
    if t.numel() != cfg.head_dim:
        raise ValueError(f"{name} must hold head_dim ({cfg.head_dim}) gains, got {tuple(t.shape)}")
    return _t(name, t, dev, _F32)


def _gpu(name, t):
    """The GPU that a call's first tensor is on: every other operand has to be there."""
    dev = t.get_device()
    if dev < 0:
        raise ValueError(f"{name} must be a device tensor")
    return dev


def _launch(dev, fn, *args):
    """fn(*args, stream) with GPU dev current (the kernels launch there), on its current stream."""
    if dev == torch._C._cuda_getDevice():
        return fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    with torch.cuda.device(dev):
        return fn(*args, torch._C._cuda_getCurrentRawStream(dev))


def _table(dev, page_table, key_len, n_pages, page, max_key_len, rope_cos=None):
    """What g4a_paged holds behind the pages, of a call's checked table and lengths."""
    if page_table.get_device() != dev or page_table.dtype is not _I32 or page_table.dim() != 2:
        raise ValueError(f"page_table must be an int32 tensor [n_seq][cols] on cuda:{dev}")
    n_seq, cols = page_table.shape
    if cols > 1 and page_table.stride(1) != 1:
        raise ValueError("page_table's columns must be adjacent")
    stride = page_table.stride(0) if n_seq > 1 else cols
    if stride < cols:
        raise ValueError("page_table rows must not overlap")
    if stride > _I32_MAX or n_seq > _I32_MAX:  # the library's struct holds 32 bits
        raise ValueError(f"page_table's rows lie too far apart, or are too many ({n_seq} rows, {stride} entries apart)")
    lens = _t("key_len", key_len, dev, _I32)
    if key_len.numel() != n_seq:
        raise ValueError(f"key_len must have one entry per row of page_table ({n_seq}), got {key_len.numel()}")
    if max_key_len is None:
        max_key_len = cols * page
        if rope_cos is not None:
            max_key_len = min(max_key_len, rope_cos.shape[0])
    if not 0 < max_key_len <= cols * page:
        raise ValueError(f"max_key_len must be in [1, {cols * page}], what the page table's columns hold")
    return page_table.data_ptr(), lens, n_pages, page, n_seq, cols, stride, int(max_key_len)


def _cache(dev, k_pages, v_pages, page_table, key_len, cfg, max_key_len, rope_cos, rope_sin):
    """The checked g4a_paged of a call, and the addresses of the RoPE tables."""
    shape, kv = k_pages.shape, k_pages.dtype
    if len(shape) != 4 or shape[2] != cfg.n_kv_heads or shape[3] != cfg.head_dim or v_pages.shape != shape:
        raise ValueError(f"k_pages / v_pages must be [n_pages][page_size][{cfg.n_kv_heads}][{cfg.head_dim}], got "
                         f"{tuple(shape)} and {tuple(v_pages.shape)}")
    if kv not in _HALF_OR_FLOAT or v_pages.dtype is not kv:
        raise ValueError("k/v pages must both be float16 or both float32")
    table = _table(dev, page_table, key_len, shape[0], shape[1], max_key_len, rope_cos)
    max_key_len = table[-1]
    if (rope_cos is None) != (rope_sin is None):
        raise ValueError("rope_cos and rope_sin go together")
    rc = rs = None
    if rope_cos is not None:
        rc, rs = _t("rope_cos", rope_cos, dev, _F32), _t("rope_sin", rope_sin, dev, _F32)
        rows = rope_cos.shape
        if len(rows) != 2 or rows[0] < max_key_len or rows[1] * 2 != cfg.head_dim or rope_sin.shape != rows:
            raise ValueError(f"rope tables must be [>= max_key_len ({max_key_len})][head_dim/2], got "
                             f"{tuple(rows)} and {tuple(rope_sin.shape)}")
    return G4APaged(_t("k_pages", k_pages, dev, kv), _t("v_pages", v_pages, dev, kv), *table), rc, rs


def _cu(cu_q, n_seq, dev):
    at = _t("cu_q", cu_q, dev, _I32)
    if cu_q.numel() != n_seq + 1:
        raise ValueError(f"cu_q must have n_seq + 1 = {n_seq + 1} entries, got {cu_q.numel()}")
    return at


def _scratch(workspace, dev, nbytes):
    """A workspace of at least nbytes on GPU dev."""
    ws = (workspace if workspace is not None else DecodeWorkspace(torch.device("cuda", dev))).get(nbytes)
    if ws.get_device() != dev:
        raise ValueError(f"workspace is on {ws.device}, the other operands on cuda:{dev}")
    return ws


def _with_scratch(workspace, dev, ws_bytes, call):
    """call(address, bytes) on the workspace's buffer; only a call that finds it too small asks for the size."""
    buf = workspace.buf if workspace is not None else None
    if buf is not None:
        if buf.get_device() != dev:
            raise ValueError(f"workspace is on {buf.device}, the other operands on cuda:{dev}")
        rc = call(buf.data_ptr(), buf.numel())
        if rc != _EWORKSPACE:
            check(rc)
            return
    need = ws_bytes()
    if need == 0:
        check(-1)
    ws = _scratch(workspace, dev, need)
    check(call(ws.data_ptr(), ws.numel()))


def paged_write(k, v, k_pages, v_pages, page_table, key_len, cu_q, cfg: AttnConfig, *, k_gain=None, rope_cos=None,
                rope_sin=None, k_in_q: float = 0.0, v_in_q: float = 0.0, v_norm: bool = True,
                max_key_len: int | None = None):
    """Append packed tokens' k/v rows ([T][kvH][hd], f32 or f16) to the cache.

    Each row is prepared as ``kv_write`` prepares it, to the bit: srq with k_in_q / v_in_q,
    k RMSNorm * k_gain and RoPE at its position, v RMSNorm."""
    if k.dim() != 3 or k.shape[1:] != (cfg.n_kv_heads, cfg.head_dim) or v.shape != k.shape or k.dtype != v.dtype:
        raise ValueError(f"k/v shape {tuple(k.shape)} does not match {cfg}")
    dev, rows = _gpu("k", k), k.dtype
    if rows not in _HALF_OR_FLOAT:
        raise ValueError(f"k and v must be float16 or float32, got {rows}")
    pg, rc, rs = _cache(dev, k_pages, v_pages, page_table, key_len, cfg, max_key_len, rope_cos, rope_sin)
    cu, kp, vp, kg = _cu(cu_q, pg.n_seq, dev), _t("k", k, dev, rows), _t("v", v, dev, rows), _gain("k_gain", k_gain, dev, cfg)
    if k.shape[0] == 0:
        return
    c = cfg.c_ref((_lib.KV_F32 if k_pages.dtype is _F32 else 0) | (_lib.IN_F16 if rows is _F16 else 0) |
                  (0 if v_norm else _lib.NO_V_NORM))
    check(_launch(dev, _lib.load().g4a_paged_write, c, ctypes.byref(pg), k.shape[0], cu, kp, vp, float(k_in_q), float(v_in_q),
                  kg, rc, rs))


def _out(out, q, out_dtype, dev):
    if out is None:
        if out_dtype not in _HALF_OR_FLOAT:
            raise ValueError(f"out_dtype must be float16 or float32, got {out_dtype}")
        out = torch.empty_like(q, dtype=out_dtype)
    elif out.shape != q.shape:
        raise ValueError(f"out must be shaped like q {tuple(q.shape)}, got {tuple(out.shape)}")
    elif out.get_device() != dev or out.dtype not in _HALF_OR_FLOAT or not out.is_contiguous():
        _refuse("out", out, dev, _HALF_OR_FLOAT)
    return out


def _q(q, cfg, q_gain):
    shape = q.shape
    if len(shape) != 3 or shape[1] != cfg.n_q_heads or shape[2] != cfg.head_dim:
        raise ValueError(f"q shape {tuple(shape)} does not match {cfg}")
    dev = _gpu("q", q)
    return dev, _t("q", q, dev, _F32), _gain("q_gain", q_gain, dev, cfg)


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
    rows are zeros. q, and K of f32 caches, keep f32 accuracy (f16 pairs); V of f32 caches is
    rounded to f16 for its product, so values beyond 65504 are infinite there.
    `workspace`: the caller's scratch (paged_decode_ws_bytes)."""
    dev, qp, qg = _q(q, cfg, q_gain)
    pg, rc, rs = _cache(dev, k_pages, v_pages, page_table, key_len, cfg, max_key_len, rope_cos, rope_sin)
    if q.shape[0] != pg.n_seq:
        raise ValueError(f"q holds {q.shape[0]} tokens, page_table {pg.n_seq} sequences")
    kn = vn = kg = None
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new go together")
    if k_new is not None:
        kn, vn, kg = _t("k_new", k_new, dev, _F32), _t("v_new", v_new, dev, _F32), _gain("k_gain", k_gain, dev, cfg)
        if k_new.shape != (pg.n_seq, cfg.n_kv_heads, cfg.head_dim) or v_new.shape != k_new.shape:
            raise ValueError(f"k_new and v_new must be [{pg.n_seq}][{cfg.n_kv_heads}][{cfg.head_dim}]")
    out = _out(out, q, out_dtype, dev)
    if pg.n_seq == 0:
        return out
    k_in_q, v_in_q = float(k_in_q), float(v_in_q)
    c = cfg.c_ref((_lib.KV_F32 if k_pages.dtype is _F32 else 0) | (_lib.OUT_F32 if out.dtype is _F32 else 0) |
                  (0 if v_norm else _lib.NO_V_NORM))
    lib, at, p = _lib.load(), out.data_ptr(), ctypes.byref(pg)
    _with_scratch(workspace, dev, lambda: lib.g4a_paged_decode_ws_bytes(c, p),
                  lambda ws, n: _launch(dev, lib.g4a_paged_decode, c, p, qp, qg, rc, rs, kn, vn, k_in_q, v_in_q, kg, at, ws, n))
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
    workspace (values beyond 65504 become infinite). `workspace`: the caller's scratch
    (paged_prefill_ws_bytes)."""
    dev, qp, qg = _q(q, cfg, q_gain)
    pg, rc, rs = _cache(dev, k_pages, v_pages, page_table, key_len, cfg, max_key_len, rope_cos, rope_sin)
    cu, n = _cu(cu_q, pg.n_seq, dev), q.shape[0]
    out = _out(out, q, out_dtype, dev)
    if n == 0:
        return out
    c = cfg.c_ref((_lib.KV_F32 if k_pages.dtype is _F32 else 0) | (_lib.OUT_F32 if out.dtype is _F32 else 0))
    lib, at, p = _lib.load(), out.data_ptr(), ctypes.byref(pg)
    _with_scratch(workspace, dev, lambda: lib.g4a_paged_prefill_ws_bytes(c, p, n),
                  lambda ws, nb: _launch(dev, lib.g4a_paged_prefill, c, p, n, cu, qp, qg, rc, rs, at, ws, nb))
    return out
