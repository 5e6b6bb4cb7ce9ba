"""The paged cache's operators, as cases that can be timed and checked: appending rows of a
ragged batch, the attention of one new token per sequence, and the attention of packed prompts.

Head counts, head sizes, the window and the RoPE bases are those of bench.py and the tests;
page sizes and batch shapes are generic serving ones. A cache holds pages [n_pages][page_size]
[kv_heads][head_dim] of K and of V in one shuffled pool for all sequences; page_table [seqs][cols]
names a sequence's pages in order. Pages behind a sliding window are given back (entry -1).
Where `own` is false the operators run in elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
NH, WINDOW, EPS = 8, 512, 1e-6
GAIN = 0.4  # mean of the q and k norm gains: scores of a few units' spread at scale 1


def listed():
    return [
        # a server's decode step appends one row per sequence: the smallest call, launches and latency
        dict(name="write_step", kind="write", seqs=16, new_min=1, new_max=1, hist_min=20, hist_max=4000, kv_heads=1,
             head_dim=256, page=16, kv="f16", rows="f32", idle=False, pad=0),
        # a batch of prompts of all lengths, the 512-wide heads of a global layer
        dict(name="write_prompts", kind="write", seqs=9, new_min=1, new_max=1111, hist_min=0, hist_max=700, kv_heads=1,
             head_dim=512, page=32, kv="f16", rows="f16", idle=False, pad=5),
        # long prompts into an f32 cache
        dict(name="write_long", kind="write", seqs=3, new_min=2000, new_max=7001, hist_min=0, hist_max=999, kv_heads=2,
             head_dim=256, page=64, kv="f32", rows="f16", idle=False, pad=0),
        # one short chat's token, its row appended: latency
        dict(name="decode_one", kind="decode", seqs=1, t_min=300, t_max=300, kv_heads=2, head_dim=256, window=0,
             page=16, kv="f16", append=True, idle=False),
        # many chats at a sliding layer, some idle; pages behind the window given back
        dict(name="decode_window", kind="decode", seqs=64, t_min=20, t_max=4097, kv_heads=1, head_dim=256,
             window=WINDOW, page=16, kv="f16", append=True, idle=True),
        # a server's batch at a global layer of 512-wide heads
        dict(name="decode_hd512", kind="decode", seqs=8, t_min=500, t_max=8200, kv_heads=1, head_dim=512, window=0,
             page=32, kv="f16", append=True, idle=False),
        # a few sequences in an f32 cache
        dict(name="decode_f32", kind="decode", seqs=4, t_min=1000, t_max=6000, kv_heads=2, head_dim=256, window=0,
             page=64, kv="f32", append=False, idle=False),
        # long contexts, ragged: the bandwidth of the card
        dict(name="decode_long", kind="decode", seqs=16, t_min=1024, t_max=32768, kv_heads=2, head_dim=256, window=0,
             page=64, kv="f16", append=False, idle=False),
        # a few short chat prompts at a sliding layer
        dict(name="prefill_chat", kind="prefill", seqs=6, new_min=5, new_max=301, hist_min=0, hist_max=0, kv_heads=1,
             head_dim=256, window=WINDOW, page=16, kv="f16", idle=False, pad=0),
        # prompts of all lengths, some continuing a cached one, at a global layer
        dict(name="prefill_mixed", kind="prefill", seqs=8, new_min=64, new_max=1900, hist_min=0, hist_max=1100,
             kv_heads=2, head_dim=256, window=0, page=64, kv="f16", idle=False, pad=7),
        # one long prompt's piece beside short ones, a sliding layer
        dict(name="prefill_window", kind="prefill", seqs=5, new_min=100, new_max=6001, hist_min=0, hist_max=2000,
             kv_heads=2, head_dim=256, window=WINDOW, page=32, kv="f16", idle=False, pad=0),
        # long prompts, 512-wide heads
        dict(name="prefill_hd512", kind="prefill", seqs=3, new_min=1000, new_max=8000, hist_min=0, hist_max=0,
             kv_heads=1, head_dim=512, window=0, page=128, kv="f16", idle=False, pad=0),
    ]


def _log(rng, lo, hi):
    """A whole number, its logarithm uniform; odd ones as often as not."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "write", "decode", "decode", "decode", "prefill", "prefill", "prefill"])
    hd = rng.choice([256, 256, 512])
    kvh = rng.choice([1, 2, 2, 4, 8]) if hd == 256 else rng.choice([1, 1, 2])
    page = rng.choice([16, 32, 64, 128])
    idle = rng.random() < 0.25
    if kind == "write":
        kvh = min(kvh, 2)
        seqs = rng.choice([1, 2, 5, 16, 33])
        new = _log(rng, 1, 14000 // (seqs * kvh * hd // 256))
        return dict(kind=kind, seqs=seqs, new_min=max(1, new // rng.choice([1, 7, 100])), new_max=new, hist_min=0,
                    hist_max=_log(rng, 1, 2000), kv_heads=kvh, head_dim=hd, page=page, kv=rng.choice(["f16", "f16", "f32"]),
                    rows=rng.choice(["f16", "f32"]), idle=idle, pad=rng.choice([0, 0, 3]))
    window = rng.choice([0, 0, WINDOW])
    if kind == "decode":
        seqs = rng.choice([1, 2, 3, 8, 16, 37, 64])
        t_max = _log(rng, 1, min(32768, 400000 // (seqs * kvh * hd // 256)))
        return dict(kind=kind, seqs=seqs, t_min=max(1, t_max // rng.choice([1, 4, 32])), t_max=t_max, kv_heads=kvh,
                    head_dim=hd, window=window, page=page,
                    kv=rng.choice(["f16", "f16", "f16", "f32"]) if seqs * t_max * kvh <= 50000 else "f16",
                    append=rng.random() < 0.6, idle=idle)
    seqs = rng.choice([1, 2, 3, 6, 12, 32])
    new = _log(rng, 1, {1: 7000, 2: 6000, 3: 5000, 6: 3500, 12: 2000, 32: 800}[seqs])
    hist = rng.choice([0, 0, _log(rng, 1, 2000)])
    return dict(kind=kind, seqs=seqs, new_min=max(1, new // rng.choice([1, 5, 60])), new_max=new, hist_min=0, hist_max=hist,
                kv_heads=kvh, head_dim=hd, window=window, page=page, kv="f16" if new > 2000 else rng.choice(["f16", "f16", "f32"]),
                idle=idle, pad=rng.choice([0, 0, 9]))


# ---------------------------------------------------------------- inputs
def _spread(n, lo, hi):
    """n whole numbers spread evenly over [lo, hi], not in order of size."""
    v = [round(lo + (hi - lo) * i / max(1, n - 1)) for i in range(n)] if n > 1 else [hi]
    return [v[(5 * i) % n] for i in range(n)] if n % 5 else v


def _lens(case):
    """(new tokens, keys) of each sequence; an idle batch has every fifth one empty."""
    n = case["seqs"]
    if case["kind"] == "decode":
        keys = _spread(n, case["t_min"], case["t_max"])
        new = [1] * n
    else:
        new = _spread(n, case["new_min"], case["new_max"])
        hist = _spread(n, case["hist_min"], case["hist_max"])[::-1]
        keys = [a + b for a, b in zip(new, hist)]
    if case["idle"]:
        for i in range(1, n, 5):
            new[i] = keys[i] = 0
    return new, keys


def _first(case, new, keys):
    """The first position of a sequence that a token of the call attends."""
    w = case.get("window", 0)
    return max(0, keys - new + 1 - w) if w else 0


def _type(name):
    return torch.float16 if name == "f16" else torch.float32


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=DEV, generator=g, dtype=dtype)

    kind, hd, kvh, page, n = case["kind"], case["head_dim"], case["kv_heads"], case["page"], case["seqs"]
    window = case.get("window", 0)
    new, keys = _lens(case)
    t_max = max(1, max(keys))
    cols = -(-t_max // page) + 1
    # pages of a shuffled pool; a few spare ones hold other sequences' rows
    table = np.full((n, cols), -1, np.int32)
    used = 0
    for b in range(n):
        lo = _first(case, new[b], keys[b]) // page
        hi = -(-keys[b] // page)
        table[b, lo:hi] = np.arange(used, used + max(0, hi - lo))
        used += max(0, hi - lo)
    n_pages = used + 3
    perm = torch.randperm(n_pages, device=DEV, generator=g)
    tab = torch.from_numpy(table).to(DEV)
    tab = torch.where(tab >= 0, perm[tab.clamp(min=0).long()].to(torch.int32), tab)
    kv = _type(case["kv"])
    state = dict(kind=kind, hd=hd, kvh=kvh, page=page, window=window, seqs=n, t_max=t_max, table=tab,
                 k_pages=(randn(n_pages, page, kvh, hd) * GAIN).to(kv), v_pages=randn(n_pages, page, kvh, hd).to(kv),
                 key_len=torch.tensor(keys, dtype=torch.int32, device=DEV), q_max=max(1, max(new)),
                 q_gain=GAIN * (1 + 0.1 * randn(hd)), k_gain=GAIN * (1 + 0.1 * randn(hd)), steps=(0.0, 0.0))
    # RoPE tables by absolute position, made in 64 bits: 1e4 at sliding layers, 1e6 at global ones
    half = hd // 2
    inv = (1e4 if window else 1e6) ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    ang = torch.arange(t_max, dtype=torch.float64, device=DEV)[:, None] * inv
    state["cos"], state["sin"] = ang.cos().float(), ang.sin().float()
    if kind == "decode":
        state["q"] = randn(n, NH, hd)
        state["append"] = case["append"]
        if case["append"]:
            state["k_new"], state["v_new"] = randn(n, kvh, hd), randn(n, kvh, hd)
        live = [b for b in range(n) if keys[b]]
        state["tok"] = live  # the rows of sequences that are not idle
    else:
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        tokens = int(cu[-1])
        state["cu"] = torch.from_numpy(cu).to(DEV)
        state["tokens"] = tokens
        rows = max(1, tokens + case["pad"])  # rows behind the last sequence belong to nobody
        if kind == "write":
            state["k_new"], state["v_new"] = (randn(rows, kvh, hd).to(_type(case["rows"])) for _ in range(2))
            # a projection's f16 rows carry its quantisation steps (steps whose borders are the same in 32 and 64 bits)
            state["steps"] = (0.0625, 0.046875) if case["rows"] == "f16" else (0.0, 0.0)
        else:
            state["q"] = randn(rows, NH, hd)
            state["out"] = torch.zeros(rows, NH, hd, dtype=torch.float16, device=DEV)
    if kind == "decode":
        state["tok"] = torch.tensor(state["tok"], dtype=torch.long, device=DEV)
    if own:
        import slang_amd as sa
        state["cfg"] = sa.AttnConfig(NH, kvh, hd, window)
        state["ws"] = sa.Workspace()
    return state


# ---------------------------------------------------------------- the plain forms
def _rms(x):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)


def _srq(x, step):
    return x if step == 0 else torch.clamp(torch.round(x / step), -128, 127) * step


def _rot(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _append(s, b, pos, k, v):
    """k and v rows of (sequence, position) pairs into their pages."""
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    k = _rot(_rms(_srq(k.float(), s["steps"][0])) * s["k_gain"], cos, sin)
    v = _rms(_srq(v.float(), s["steps"][1]))
    at = s["table"][b, pos // s["page"]].long() * s["page"] + pos % s["page"]
    s["k_pages"].view(-1, s["kvh"], s["hd"])[at] = k.to(s["k_pages"].dtype)
    s["v_pages"].view(-1, s["kvh"], s["hd"])[at] = v.to(s["v_pages"].dtype)


def _attend(s, q, pos):
    """q [n][S][nH][hd], normed and rotated, at positions pos [n][S] (below zero: no token): f16 outputs."""
    n, S, kvh, hd = q.shape[0], q.shape[1], s["kvh"], s["hd"]
    T = s["t_max"]
    idx = s["table"][:, :-(-T // s["page"])].clamp(min=0).long()
    k = s["k_pages"][idx].flatten(1, 2)[:, :T].float()  # [n][T][kvH][hd]
    v = s["v_pages"][idx].flatten(1, 2)[:, :T].float()
    q = q.reshape(n, S, kvh, NH // kvh, hd).permute(0, 2, 3, 1, 4).reshape(n, kvh, (NH // kvh) * S, hd)
    sc = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(n, kvh, NH // kvh, S, T)
    t = torch.arange(T, device=DEV)
    seen = t <= pos[..., None]
    if s["window"]:
        seen &= t > pos[..., None] - s["window"]
    seen = seen[:, None, None]
    sc = sc.masked_fill_(~seen, float("-inf"))
    p = torch.exp_(sc.sub_(sc.amax(-1, keepdim=True).clamp(min=-1e30)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, kvh, -1, T), v.permute(0, 2, 1, 3).contiguous()).view(n, kvh, NH // kvh, S, hd)
    o = torch.where(total > 0, o / total.clamp(min=1e-30), torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(n, S, NH, hd).half()


def run(s):
    kind = s["kind"]
    if own:
        import slang_amd as sa
        if kind == "write":
            sa.paged_write(s["k_new"], s["v_new"], s["k_pages"], s["v_pages"], s["table"], s["key_len"], s["cu"], s["cfg"],
                           k_gain=s["k_gain"], rope_cos=s["cos"], rope_sin=s["sin"], k_in_q=s["steps"][0],
                           v_in_q=s["steps"][1], max_key_len=s["t_max"])
            return s["k_pages"], s["v_pages"]
        if kind == "decode":
            new = dict(k_new=s["k_new"], v_new=s["v_new"], k_gain=s["k_gain"]) if s["append"] else {}
            out = sa.paged_decode(s["q"], s["k_pages"], s["v_pages"], s["table"], s["key_len"], s["cfg"],
                                  workspace=s["ws"], q_gain=s["q_gain"], rope_cos=s["cos"], rope_sin=s["sin"],
                                  max_key_len=s["t_max"], **new)
            return (out, s["k_pages"], s["v_pages"]) if s["append"] else out
        return sa.paged_prefill(s["q"], s["k_pages"], s["v_pages"], s["table"], s["key_len"], s["cu"], s["cfg"],
                                workspace=s["ws"], q_gain=s["q_gain"], rope_cos=s["cos"], rope_sin=s["sin"],
                                out=s["out"], max_key_len=s["t_max"])
    if kind == "decode":
        last = s["key_len"].long() - 1  # -1: an idle sequence
        if s["append"]:
            _append(s, s["tok"], last[s["tok"]], s["k_new"][s["tok"]], s["v_new"][s["tok"]])
        at = last.clamp(min=0)
        q = _rot(_rms(s["q"]) * s["q_gain"], s["cos"][at][:, None], s["sin"][at][:, None])
        out = _attend(s, q[:, None], last[:, None])[:, 0]
        return (out, s["k_pages"], s["v_pages"]) if s["append"] else out
    cu, key_len, tokens = s["cu"].long(), s["key_len"].long(), s["tokens"]
    tok = torch.arange(tokens, device=DEV)
    b = torch.searchsorted(cu[1:], tok, right=True)
    i = tok - cu[b]
    pos = key_len[b] - (cu[b + 1] - cu[b]) + i
    if kind == "write":
        _append(s, b, pos, s["k_new"][:tokens], s["v_new"][:tokens])
        return s["k_pages"], s["v_pages"]
    q = _rot(_rms(s["q"][:tokens]) * s["q_gain"], s["cos"][pos][:, None], s["sin"][pos][:, None])
    q_pad = torch.zeros(s["seqs"], s["q_max"], NH, s["hd"], device=DEV)
    pos_pad = torch.full((s["seqs"], s["q_max"]), -1, dtype=torch.long, device=DEV)
    q_pad[b, i] = q
    pos_pad[b, i] = pos
    s["out"][:tokens] = _attend(s, q_pad, pos_pad)[b, i]
    return s["out"]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    new, keys = _lens(case)
    hd, kvh, w = case["head_dim"], case["kv_heads"], case.get("window", 0)
    esz = 2 if case["kv"] == "f16" else 4
    row = kvh * hd
    if case["kind"] == "write":
        tokens = sum(new)
        return {"bytes": 2 * tokens * row * ((2 if case["rows"] == "f16" else 4) + esz), "flops": 10 * 2 * tokens * row}
    read = sum(k - _first(case, a, k) for a, k in zip(new, keys)) * row * 2 * esz  # each attended row once
    queries = sum(1 for k in keys if k) if case["kind"] == "decode" else sum(new)
    total = read + queries * NH * hd * (4 + 2)
    if case.get("append"):
        total += queries * row * 2 * 4
    pairs = 0
    for a, k in zip(new, keys):
        p = np.arange(k - a, k, dtype=np.int64) + 1
        pairs += int(np.minimum(p, w).sum() if w else p.sum())
    return {"bytes": total, "flops": 4 * hd * NH * pairs}


# ---------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    new, keys = _lens(case)
    hd, kvh, page, w = case["head_dim"], case["kv_heads"], case["page"], case.get("window", 0)
    table = s["table"].cpu().numpy()
    f8 = torch.float64
    cos, sin = s["cos"].to(f8), s["sin"].to(f8)

    def normed(x):
        return x * (x.pow(2).sum(-1, keepdim=True) / hd + EPS).rsqrt()

    def rotated(x, at):  # as a complex product of the pairs (i, i + hd/2)
        z = torch.complex(x[..., : hd // 2], x[..., hd // 2:]) * torch.complex(cos[at], sin[at])[:, None]
        return torch.cat((z.real, z.imag), -1)

    def stepped(x, step):
        step = float(np.float32(step))
        return (x / step).round().clamp(-128, 127) * step if step else x

    kp, vp = s["k_pages"].to(f8), s["v_pages"].to(f8)
    first, rows_of = 0, []
    for b in range(case["seqs"]):  # each sequence's rows in the pool, in order
        p = np.arange(keys[b])
        pages = table[b, p // page] if keys[b] else np.zeros(0, np.int32)
        rows_of.append(torch.from_numpy(np.where(pages < 0, 0, pages).astype(np.int64) * page + p % page).to(DEV))
    if case["kind"] == "write" or case.get("append"):
        kr, vr = kp.view(-1, kvh, hd), vp.view(-1, kvh, hd)
        for b in range(case["seqs"]):
            at = torch.arange(keys[b] - new[b], keys[b], device=DEV)
            first_b = b if case["kind"] == "decode" else first
            if new[b]:
                k = stepped(s["k_new"][first_b:first_b + new[b]].to(f8), s["steps"][0])
                v = stepped(s["v_new"][first_b:first_b + new[b]].to(f8), s["steps"][1])
                kr[rows_of[b][at]] = rotated(normed(k) * s["k_gain"].to(f8), at)
                vr[rows_of[b][at]] = normed(v)
            first += new[b]
        if case["kind"] == "write":
            return kp, vp
    att_k, att_v = kp, vp
    if case.get("append"):  # what is attended is what the cache holds
        att_k, att_v = kp.to(s["k_pages"].dtype).to(f8), vp.to(s["v_pages"].dtype).to(f8)
    att_k, att_v = att_k.view(-1, kvh, hd), att_v.view(-1, kvh, hd)
    out = torch.zeros(s["q"].shape, dtype=f8, device=DEV)
    first = 0
    for b in range(case["seqs"]):
        first_b = b if case["kind"] == "decode" else first
        first += new[b]
        for c0 in range(0, new[b], 1024):
            at = torch.arange(keys[b] - new[b] + c0, keys[b] - new[b] + min(c0 + 1024, new[b]), device=DEV)
            q = s["q"][first_b + c0:first_b + c0 + len(at)].to(f8)
            q = rotated(normed(q) * s["q_gain"].to(f8), at)
            lo = max(0, int(keys[b] - new[b] + c0 + 1 - w)) if w else 0
            hi = int(keys[b] - new[b] + c0 + len(at))
            t = torch.arange(lo, hi, device=DEV)
            off = t > at[:, None]
            if w:
                off |= at[:, None] - t >= w
            for h in range(NH):
                kh = h // (NH // kvh)
                sc = q[:, h] @ att_k[rows_of[b][lo:hi], kh].T.contiguous()
                sc[off] = float("-inf")
                out[first_b + c0:first_b + c0 + len(at), h] = torch.softmax(sc, -1) @ att_v[rows_of[b][lo:hi], kh]
    return (out, kp, vp) if case.get("append") else out
