"""Generation that branches, over the paged cache of paged.py: drafted trees and beams.

A server that drafts several continuations of a sequence checks them all in one step. The drafts of a
sequence form a tree, packed as its last rows:

  * ``parents`` int32 [T]: token i of a tree continues token ``parents[i]`` < i of the same tree, anything
    else (-1) makes it a root, which continues the sequence's last key. Token 0 is by custom the last
    sampled token, the others its drafts;
  * token i sits at row key_len - n + i of its sequence's n new rows, but at position
    key_len - n + depth(i): siblings share one.

``paged_tree`` writes the tree's k/v rows and attends.

Lengths, offsets, parents and tables stay on the GPU, so a captured graph of a step can be replayed on
new ones. Calls run on the current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import check
from .attention import AttnConfig, DecodeWorkspace
from .paged import _F16, _F32, _HALF_OR_FLOAT, _I32, _cache, _cu, _gain, _launch, _out, _q, _sizes, _t, _with_scratch

__all__ = ["paged_tree", "paged_tree_ws_bytes"]


def _parents(parents, n, dev):
    at = _t("parents", parents, dev, _I32)
    if parents.dim() != 1 or parents.shape[0] != n:
        raise ValueError(f"parents must hold one entry per packed token ({n}), got {tuple(parents.shape)}")
    return at


def paged_tree_ws_bytes(n_tokens: int, n_seq: int, max_key_len: int, cfg: AttnConfig, *, page_size: int,
                        kv_f32: bool = False) -> int:
    """Workspace bytes of a ``paged_tree`` call (g4a_paged_tree_ws_bytes): reserve the largest call's."""
    c = cfg.c(_lib.KV_F32 if kv_f32 else 0)
    pg = _sizes(1, page_size, n_seq, -(-max_key_len // page_size), max_key_len)
    n = _lib.load().g4a_paged_tree_ws_bytes(ctypes.byref(c), ctypes.byref(pg), int(n_tokens))
    if n == 0:
        check(-1)
    return int(n)


def paged_tree(q, k_pages, v_pages, page_table, key_len, cu_q, parents, cfg: AttnConfig, *, workspace: DecodeWorkspace,
               q_gain=None, rope_cos=None, rope_sin=None, k_new=None, v_new=None, k_gain=None, k_in_q: float = 0.0,
               v_in_q: float = 0.0, v_norm: bool = True, out=None, out_dtype=torch.float16, max_key_len: int | None = None):
    """Attention of packed drafted trees, a tree per sequence, over the cache.

    A token attends its sequence's keys in front of the tree, its ancestors and itself, within cfg's window
    of its position. q f32 [T][nH][hd] raw, rounded to f16 once normalised and rotated. With k_new / v_new ([T][kvH][hd],
    f32 or f16) the tokens' rows are prepared as ``kv_write`` prepares them, each at its position, and stored
    by the same call before they are attended; without, the cache holds them. A tree has at most 1024 tokens: rows
    behind are rows of nobody. Returns out [T][nH][hd] (f16 by default). f32 caches are converted to f16 in the
    workspace (values beyond 65504 become infinite). `workspace`: the caller's scratch (paged_tree_ws_bytes)."""
    dev, qp, qg = _q(q, cfg, q_gain)
    pg, rc, rs = _cache(dev, k_pages, v_pages, page_table, key_len, cfg, max_key_len, rope_cos, rope_sin)
    n = q.shape[0]
    cu, par = _cu(cu_q, pg.n_seq, dev), _parents(parents, n, dev)
    kn = vn = kg = None
    rows = _F32
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new go together")
    if k_new is not None:
        rows = k_new.dtype
        if rows not in _HALF_OR_FLOAT:
            raise ValueError(f"k_new and v_new must be float16 or float32, got {rows}")
        kn, vn, kg = _t("k_new", k_new, dev, rows), _t("v_new", v_new, dev, rows), _gain("k_gain", k_gain, dev, cfg)
        if k_new.shape != (n, cfg.n_kv_heads, cfg.head_dim) or v_new.shape != k_new.shape:
            raise ValueError(f"k_new and v_new must be [{n}][{cfg.n_kv_heads}][{cfg.head_dim}]")
    out = _out(out, q, out_dtype, dev)
    if n == 0 or pg.n_seq == 0:
        return out
    k_in_q, v_in_q = float(k_in_q), float(v_in_q)
    c = cfg.c_ref((_lib.KV_F32 if k_pages.dtype is _F32 else 0) | (_lib.OUT_F32 if out.dtype is _F32 else 0) |
                  (_lib.IN_F16 if rows is _F16 else 0) | (0 if v_norm else _lib.NO_V_NORM))
    lib, at, p = _lib.load(), out.data_ptr(), ctypes.byref(pg)
    _with_scratch(workspace, dev, lambda: lib.g4a_paged_tree_ws_bytes(c, p, n),
                  lambda ws, nb: _launch(dev, lib.g4a_paged_tree, c, p, n, cu, par, qp, qg, rc, rs, kn, vn, k_in_q, v_in_q, kg,
                                         at, ws, nb))
    return out
