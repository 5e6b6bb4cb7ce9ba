"""Generation that branches, over the paged cache of paged.py: drafted trees and beams.

A server that drafts several continuations of a sequence checks them all in one step. The drafts of a
sequence form a tree, packed as its last rows:

  * ``parents`` int32 [T]: token i of a tree continues token ``parents[i]`` < i of the same tree, anything
    else (-1) makes it a root, which continues the sequence's last key. Token 0 is by custom the last
    sampled token, the others its drafts;
  * token i sits at row key_len - n + i of its sequence's n new rows, but at position
    key_len - n + depth(i): siblings share one.

A step of a server that drafts, per layer: ``paged_tree`` stores the tree's k/v rows and attends. Then
``tree_accept`` walks the drafts that the model agrees with, and ``paged_keep`` moves their rows, in all layers
at once, to where plain steps would have put them; what lies behind is the next step's to overwrite.

Beams are rows of one page table. A step: ``beam_select`` picks the next tokens and the beams that they continue;
``paged_fork`` makes the tables that follow, in which full pages are shared, the pages that beams write to are
their own, and pages of no beam are free again.

Lengths, offsets, parents, tables and free lists stay on the GPU, so a captured graph of a step can be replayed
on new ones. Calls run on the current stream of the tensors' device.
"""
from __future__ import annotations

import array
import ctypes
import math

import torch

from . import _lib
from ._lib import G4APaged, check
from .attention import AttnConfig, DecodeWorkspace
from .paged import (_F16, _F32, _HALF_OR_FLOAT, _I32, _cache, _cu, _gain, _gpu, _launch, _out, _q, _refuse, _sizes, _t, _table,
                    _with_scratch)

__all__ = ["CachePools", "paged_tree", "paged_tree_ws_bytes", "tree_accept", "paged_keep", "paged_fork", "paged_fork_ws_bytes",
           "beam_select", "beam_select_ws_bytes"]


class CachePools:
    """The K and V pages of a cache's layers, checked once: tensors [n_pages][page_size][...] on one GPU, up to 64, whose
    rows may differ in heads, head size and type from layer to layer. The calls that take ``pools`` take one of these or a
    list of tensors, which they then check anew each time."""

    def __init__(self, pools):
        pools = self.tensors = list(pools)
        if len(pools) > _lib.POOLS_MAX:
            raise ValueError(f"at most {_lib.POOLS_MAX} pools a call, got {len(pools)}")
        self.dev, self.shape, at, like, kind, row = -1, (0, 0), [], None, None, 0
        for p in pools:
            if p.shape != like or p.dtype is not kind:  # layers are mostly alike
                like, kind = p.shape, p.dtype
                if len(like) < 3:
                    raise ValueError(f"a pool must be [n_pages][page_size][...], got {tuple(like)}")
                if not at:
                    self.dev, self.shape = _gpu("a pool", p), tuple(like[:2])
                if tuple(like[:2]) != self.shape:
                    raise ValueError(f"a pool holds {tuple(like[:2])} pages and rows, the first one {self.shape}")
                row = math.prod(like[2:]) * p.element_size()
            if p.get_device() != self.dev or not p.is_contiguous():
                _refuse("a pool", p, self.dev, kind)
            at += p.data_ptr(), row
        self._c = array.array("q", at)  # struct g4a_pool [n]: an address, bytes of a row
        self.c = self._c.buffer_info()[0]

    def __len__(self):
        return len(self.tensors)


def _pools(pools, dev):
    if not isinstance(pools, CachePools):
        pools = CachePools(pools)
    if len(pools) and pools.dev != dev:
        raise ValueError(f"the pools are on cuda:{pools.dev}, the other operands on cuda:{dev}")
    return pools


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
    of its position. q f32 [T][nH][hd] raw; normalised and rotated, it enters the products at f32 accuracy (f16
    pairs), as in ``paged_decode``, and so does K of f32 caches. With k_new / v_new ([T][kvH][hd], f32 or f16) the tokens' rows
    are prepared as ``kv_write`` prepares them, each at its position, and stored by the same call before they are
    attended; without, the cache holds them. A tree has at most 1024 tokens: rows behind are rows of nobody. Returns
    out [T][nH][hd] (f16 by default). f32 caches are converted in the workspace, K to pairs of f16 and V to f16 (values
    beyond 65504 make what attends them infinite or NaN). `workspace`: the caller's scratch (paged_tree_ws_bytes)."""
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


def _i32(name, t, dev, shape):
    at = _t(name, t, dev, _I32)
    if t.shape != shape:
        raise ValueError(f"{name} must be int32 {list(shape)}, got {tuple(t.shape)}")
    return at


def tree_accept(drafts, targets, parents, cu_q, key_len, *, max_path: int | None = None, out=None):
    """The path of drafts that the model agrees with, per sequence (greedy verification).

    drafts [T]: the packed trees' tokens; targets [T]: the token that the model puts behind each (``beam_select`` of width 1
    gives the row-wise argmax). The path is token 0, then, while there is one, the child of lowest index of the path's last
    token whose draft is that token's target. Returns int32 tensors (path [n_seq][max_path] of indices within the
    trees, -1 behind the end; n_path [n_seq]; next [n_seq], the last one's target, -1 for a sequence without tokens;
    kept [n_seq], key_len less the tokens that are not on the path). `out`: the four, made by an earlier call.
    max_path: the longest path (default: T, at most 1024); a longer one ends there."""
    dev = _gpu("drafts", drafts)
    if drafts.dim() != 1:
        raise ValueError(f"drafts must hold one token per packed row, got {tuple(drafts.shape)}")
    n, n_seq = drafts.shape[0], key_len.numel()
    dr, tg, par = _t("drafts", drafts, dev, _I32), _i32("targets", targets, dev, (n,)), _parents(parents, n, dev)
    lens, cu = _t("key_len", key_len, dev, _I32), _cu(cu_q, n_seq, dev)
    max_path = max(1, min(n, _lib.TREE_MAX)) if max_path is None else int(max_path)
    if max_path < 1:
        raise ValueError(f"max_path must be positive, got {max_path}")
    if out is None:
        one = key_len if key_len.dim() == 1 else key_len.view(-1)
        out = (torch.empty((n_seq, max_path), dtype=_I32, device=drafts.device), torch.empty_like(one), torch.empty_like(one),
               torch.empty_like(one))
        at = [t.data_ptr() for t in out]
    else:
        shapes = ((n_seq, max_path), (n_seq,), (n_seq,), (n_seq,))
        at = [_i32(name, t, dev, s) for name, t, s in zip(("path", "n_path", "next", "kept"), out, shapes)]
    if n_seq == 0:
        return tuple(out)
    if n == 0:  # no sequence has a token
        out[0].fill_(-1), out[1].zero_(), out[2].fill_(-1), out[3].copy_(key_len.view(-1))
        return tuple(out)
    check(_launch(dev, _lib.load().g4a_tree_accept, n, n_seq, cu, par, dr, tg, lens, max_path, *at))
    return tuple(out)


def paged_keep(pools, page_table, key_len, cu_q, path, n_path, *, n_tokens: int | None = None, max_key_len: int | None = None):
    """Moves the rows of accepted paths up, in every pool: row key_len - n + path[b][d] of a sequence with n tokens in its tree to
    row key_len - n + d, for d < n_path[b]. key_len and cu_q are those of the tree's call; afterwards the sequence has
    ``tree_accept``'s `kept` keys. path [n_seq][max_path] ascends in each row; it ends at an entry that does not.
    pools: a ``CachePools`` or tensors [n_pages][page_size][...], K and V of any number of layers up to 32.
    n_tokens: the packed rows of the tree's call where offsets could lead past them (default: no bound)."""
    dev = _gpu("page_table", page_table)
    pools = _pools(pools, dev)
    if not len(pools):
        return
    pg = G4APaged(None, None, *_table(dev, page_table, key_len, *pools.shape, max_key_len))
    cu = _cu(cu_q, pg.n_seq, dev)
    if path.dim() != 2 or path.shape[0] != pg.n_seq:
        raise ValueError(f"path must be int32 [{pg.n_seq}][max_path], got {tuple(path.shape)}")
    at, count = _t("path", path, dev, _I32), _i32("n_path", n_path, dev, (pg.n_seq,))
    n_tokens = 2 ** 31 - 1 if n_tokens is None else int(n_tokens)
    if pg.n_seq == 0 or path.shape[1] == 0 or n_tokens == 0:
        return
    check(_launch(dev, _lib.load().g4a_paged_keep, pools.c, len(pools), ctypes.byref(pg), n_tokens, cu, at, path.shape[1], count))


def paged_fork_ws_bytes(n_pages: int, n_new: int) -> int:
    """Workspace bytes of a ``paged_fork`` call (g4a_paged_fork_ws_bytes): reserve the largest call's."""
    pg = _sizes(n_pages, 16, 1, 1, 16)
    n = _lib.load().g4a_paged_fork_ws_bytes(ctypes.byref(pg), int(n_new))
    if n == 0:
        check(-1)
    return int(n)


def paged_fork(pools, page_table, key_len, parent, free_pages, n_free, *, workspace: DecodeWorkspace, room: int = 1, out=None,
               n_pages: int | None = None, page_size: int | None = None, max_key_len: int | None = None):
    """The tables, lengths and free list of sequences that follow their parents (beams after a step's selection).

    New row j continues row parent[j] (int32, n_new of them in any shape) of page_table [n_seq][cols], which lists every
    sequence that has pages of the pools (one that does not branch is its own parent; a parent outside [0, n_seq) makes
    an idle row). Full pages are shared; each page that a row will write to, for `room` more keys, becomes its own: the
    first heir keeps the parent's, the others get pages off the end of free_pages (int32 [n_pages], its first n_free
    (int32 [1]) are free), and the filled rows of a partly filled one are copied in every pool. Pages that no new row
    holds are added to the list first, in order.
    Returns (table [n_new][cols], key_len [n_new], free_pages, n_free), all new tensors, or the four given as `out` (none of
    them an input: alternate two sets in a captured loop). Too few free pages leave -1 in the last columns that need one;
    n_new * (2 + room // page_size) always suffice. n_pages and page_size are needed where there are no pools.
    `workspace`: the caller's scratch (paged_fork_ws_bytes)."""
    dev = _gpu("page_table", page_table)
    pools = _pools(pools, dev)
    shape = pools.shape if len(pools) else (n_pages, page_size)
    if None in shape or n_pages not in (None, shape[0]) or page_size not in (None, shape[1]):
        raise ValueError(f"n_pages ({n_pages}) and page_size ({page_size}) must be those of the pools, {tuple(shape)}")
    pg = G4APaged(None, None, *_table(dev, page_table, key_len, *shape, max_key_len))
    n_new, par = parent.numel(), _t("parent", parent, dev, _I32)
    fr, nf = _i32("free_pages", free_pages, dev, (pg.n_pages,)), _i32("n_free", n_free, dev, (1,))
    room = int(room)
    if not 0 <= room <= 1 << 30:
        raise ValueError(f"room must be in [0, 2^30], got {room}")
    if out is None:
        out = (torch.empty((n_new, pg.table_cols), dtype=_I32, device=page_table.device), torch.empty_like(parent.view(-1)),
               torch.empty_like(free_pages), torch.empty_like(n_free))
        at = [t.data_ptr() for t in out]
    else:
        shapes = ((n_new, pg.table_cols), (n_new,), (pg.n_pages,), (1,))
        at = [_i32(name, t, dev, s) for name, t, s in zip(("new table", "new key_len", "new free_pages", "new n_free"), out, shapes)]
    if pg.n_seq == 0 or n_new == 0:
        raise ValueError("paged_fork needs a row to follow and a row that follows")
    lib, p = _lib.load(), ctypes.byref(pg)
    _with_scratch(workspace, dev, lambda: lib.g4a_paged_fork_ws_bytes(p, n_new),
                  lambda ws, nb: _launch(dev, lib.g4a_paged_fork, pools.c, len(pools), p, n_new, par, room, fr, nf, *at, ws, nb))
    return tuple(out)


def beam_select_ws_bytes(n_groups: int, width: int, vocab: int, n_out: int | None = None) -> int:
    """Workspace bytes of a ``beam_select`` call (g4a_beam_select_ws_bytes)."""
    n = _lib.load().g4a_beam_select_ws_bytes(int(n_groups), int(width), int(vocab), int(width if n_out is None else n_out))
    if n == 0:
        check(-1)
    return int(n)


def beam_select(logits, scores, *, workspace: DecodeWorkspace, cap: float = 0.0, n_out: int | None = None, done=None, pad: int = 0,
                out=None):
    """The n_out best continuations of each group of beams (default: as many as beams).

    logits f32 or f16 [n_groups * width][V], 16-byte aligned (rows may lie further apart than V); scores f32
    [n_groups][width]: the beams' sums of log probabilities. A candidate scores its beam's plus log softmax(cap *
    tanh(logits / cap)) (cap 0: of the logits). done (bool [n_groups][width]): a finished beam has one candidate, token
    `pad` at its own score. Logits of -inf or NaN are no tokens. Returns (score f32, parent int32, token int32), each
    [n_groups][n_out], best first: a beam's candidates in the order of their logits (a cap moves none of them), equal
    logits by token, equal scores of two beams by beam; parent is the row of logits, which ``paged_fork`` takes as it
    is. Places that no candidate of a score above -inf fills hold -inf, -1, -1. At most 64 beams, 64 places, 65535 rows of
    logits. `out`: the three, made by an earlier call. `workspace`: the caller's scratch (beam_select_ws_bytes)."""
    if scores.dim() != 2:
        raise ValueError(f"scores must be [n_groups][width], got {tuple(scores.shape)}")
    dev, (groups, width) = _gpu("logits", logits), scores.shape
    if logits.dtype not in _HALF_OR_FLOAT or logits.dim() != 2 or logits.shape[0] != groups * width:
        raise ValueError(f"logits must be float16 or float32 [{groups * width}][V], got {logits.dtype} {tuple(logits.shape)}")
    vocab = logits.shape[1]
    stride = logits.stride(0) if logits.shape[0] > 1 else max(vocab, 1)
    if vocab > 1 and logits.stride(1) != 1 or stride < vocab:
        raise ValueError("a row's logits must be adjacent, and rows must not overlap")
    sc = _t("scores", scores, dev, _F32)
    n_out = width if n_out is None else int(n_out)
    dn = None
    if done is not None:
        if done.shape != scores.shape or done.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"done must be bool, shaped like scores {tuple(scores.shape)}, got {done.dtype} {tuple(done.shape)}")
        dn = _t("done", done, dev, done.dtype)
    if out is None:
        where = logits.device
        if n_out < 0:
            raise ValueError(f"n_out must be positive, got {n_out}")
        token = torch.empty((groups, n_out), dtype=_I32, device=where)
        out = torch.empty((groups, n_out), dtype=_F32, device=where), torch.empty_like(token), token
        at = [t.data_ptr() for t in out]
    else:
        at = []
        for name, t, kind in zip(("score", "parent", "token"), out, (_F32, _I32, _I32)):
            at.append(_t(name, t, dev, kind))
            if tuple(t.shape) != (groups, n_out):
                raise ValueError(f"{name} must be [{groups}][{n_out}], got {tuple(t.shape)}")
    if groups == 0:
        return tuple(out)
    lib, f16 = _lib.load(), int(logits.dtype is _F16)
    pad, cap = int(pad), float(cap)
    _with_scratch(workspace, dev, lambda: lib.g4a_beam_select_ws_bytes(groups, width, vocab, n_out),
                  lambda ws, nb: _launch(dev, lib.g4a_beam_select, groups, width, vocab, f16, logits.data_ptr(), stride, sc, dn, pad, cap,
                                         n_out, *at, ws, nb))
    return tuple(out)
