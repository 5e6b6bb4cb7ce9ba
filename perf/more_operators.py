"""The operators of generation that branches over the paged cache, as cases that can be timed and
checked: the attention of a tree of drafted tokens, the walk that accepts drafts, moving the
accepted rows up, beam search's selection, and the fork of page tables that follows it.

Head counts, head sizes, the window, the RoPE bases, the softcap and the vocabulary are those of
bench.py and the tests; page sizes and batch shapes are generic serving ones. Caches are pages
[n_pages][page_size][kv_heads][head_dim] of K and of V in one shuffled pool for all sequences,
page_table [seqs][cols] names a sequence's pages in order (-1: not there). A tree's token i sits at
row key_len - n + i of its sequence, at position key_len - n + depth(i); its parent has a lower index.
Where `own` is false the operators run in elementary torch operations in 32 bits (a beam's
scores, which decide over whole numbers, in 64).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
NH, WINDOW, EPS, CAP, VOCAB = 8, 512, 1e-6, 30.0, 262144
GAIN = 0.4  # mean of the q and k norm gains: scores of a few units' spread at scale 1


def listed():
    return [
        # one chat's drafts: the smallest call, launches and latency
        dict(name="tree_one", kind="tree", seqs=1, tree_min=12, tree_max=12, hist_min=300, hist_max=300, kv_heads=2,
             head_dim=256, window=0, page=16, kv="f16", append=True, idle=False, pad=0),
        # many chats' drafts at a sliding layer, some idle; pages behind the window given back
        dict(name="tree_window", kind="tree", seqs=32, tree_min=1, tree_max=33, hist_min=20, hist_max=4000, kv_heads=1,
             head_dim=256, window=WINDOW, page=16, kv="f16", append=True, idle=True, pad=3),
        # wide trees over an f32 cache of 512-wide heads
        dict(name="tree_wide", kind="tree", seqs=3, tree_min=60, tree_max=253, hist_min=500, hist_max=5000, kv_heads=1,
             head_dim=512, window=0, page=32, kv="f32", append=True, idle=False, pad=0),
        # long contexts, ragged: the bandwidth of the card
        dict(name="tree_long", kind="tree", seqs=16, tree_min=5, tree_max=40, hist_min=1024, hist_max=32768, kv_heads=2,
             head_dim=256, window=0, page=64, kv="f16", append=False, idle=False, pad=0),
        # one chat's drafts walked: latency
        dict(name="accept_one", kind="accept", seqs=1, tree_min=12, tree_max=12, hist_min=300, hist_max=300, idle=False, pad=0),
        # a server's batch of wide trees, some idle
        dict(name="accept_batch", kind="accept", seqs=200, tree_min=1, tree_max=253, hist_min=0, hist_max=4000, idle=True, pad=5),
        # one layer's rows of a few accepted paths
        dict(name="keep_layer", kind="keep", seqs=4, tree_min=6, tree_max=40, hist_min=20, hist_max=900, kv_heads=1,
             head_dim=256, page=16, kv="f16", layers=1, idle=False, pad=0),
        # all layers' rows of a batch's accepted paths
        dict(name="keep_layers", kind="keep", seqs=32, tree_min=8, tree_max=64, hist_min=0, hist_max=300, kv_heads=2,
             head_dim=256, page=32, kv="f16", layers=15, idle=True, pad=2),
        # one sequence's beams over a small vocabulary: latency
        dict(name="beam_one", kind="beam", groups=1, beams=4, vocab=32000, out=4, logits="f32", cap=0.0, first=False, done=False),
        # a batch of beams over the whole vocabulary, some finished: the bandwidth of the card
        dict(name="beam_batch", kind="beam", groups=16, beams=8, vocab=VOCAB, out=16, logits="f32", cap=CAP, first=False, done=True),
        # one sequence's beams fork: the smallest call
        dict(name="fork_one", kind="fork", groups=1, beams=4, prompt_min=100, prompt_max=100, grown_min=5, grown_max=60, kv_heads=1,
             head_dim=256, page=16, kv="f16", layers=1, room=1),
        # a batch's beams in all layers
        dict(name="fork_layers", kind="fork", groups=16, beams=8, prompt_min=10, prompt_max=2000, grown_min=1, grown_max=300,
             kv_heads=1, head_dim=256, page=32, kv="f16", layers=15, room=1),
    ]


def _log(rng, lo, hi):
    """A whole number, its logarithm uniform; odd ones as often as not."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "tree", "accept", "keep", "beam", "beam", "fork"])
    hd = rng.choice([256, 256, 512])
    kvh = rng.choice([1, 2, 2, 4, 8]) if hd == 256 else rng.choice([1, 1, 2])
    page = rng.choice([16, 32, 64, 128])
    idle = rng.random() < 0.25
    if kind == "beam":
        groups, beams = rng.choice([1, 2, 5, 16]), rng.choice([1, 2, 4, 5, 8])
        vocab = _log(rng, 500, VOCAB)
        return dict(kind=kind, groups=groups, beams=beams, vocab=vocab, out=beams * rng.choice([1, 2]),
                    logits=rng.choice(["f32", "f32", "f16"]), cap=rng.choice([0.0, CAP]), first=rng.random() < 0.2,
                    done=rng.random() < 0.4)
    if kind == "fork":
        groups, beams, layers = rng.choice([1, 2, 7, 16]), rng.choice([1, 2, 4, 8]), rng.choice([1, 3, 15])
        prompt, grown = _log(rng, 1, 2000), _log(rng, 1, 300)
        kvh = min(kvh, 2) if layers < 15 else 1
        return dict(kind=kind, groups=groups, beams=beams, prompt_min=max(1, prompt // rng.choice([1, 5])), prompt_max=prompt,
                    grown_min=max(1, grown // rng.choice([1, 9])), grown_max=grown, kv_heads=kvh, head_dim=256, page=min(page, 64),
                    kv=rng.choice(["f16", "f16", "f32"]) if layers < 15 else "f16", layers=layers, room=rng.choice([1, 1, 7]))
    seqs = rng.choice([1, 2, 5, 16, 33])
    if kind == "accept":
        tree = _log(rng, 1, 253)
        return dict(kind=kind, seqs=seqs, tree_min=max(1, tree // rng.choice([1, 3, 20])), tree_max=tree, hist_min=0,
                    hist_max=_log(rng, 1, 4000), idle=idle, pad=rng.choice([0, 0, 3]))
    if kind == "keep":
        tree, layers = _log(rng, 2, 100), rng.choice([1, 3, 15])
        return dict(kind=kind, seqs=seqs, tree_min=max(1, tree // rng.choice([1, 3])), tree_max=tree, hist_min=0,
                    hist_max=_log(rng, 1, 300), kv_heads=min(kvh, 2), head_dim=hd if layers < 15 else 256, page=page,
                    kv=rng.choice(["f16", "f16", "f32"]) if layers < 15 else "f16", layers=layers, idle=idle, pad=rng.choice([0, 0, 3]))
    window = rng.choice([0, 0, WINDOW])
    kv = rng.choice(["f16", "f16", "f16", "f32"])
    # the plain form works over all pairs of a padded batch: at most those of the largest listed case
    tree = _log(rng, 1, max(1, min(253, 640 // seqs)))
    most = int(min(32768, 16 * 32768 * 2 * 256 / (seqs * kvh * hd * (2 if kv == "f32" else 1))))
    hist = _log(rng, 16, most)
    return dict(kind=kind, seqs=seqs, tree_min=max(1, tree // rng.choice([1, 2, 8])), tree_max=tree,
                hist_min=hist // rng.choice([1, 2, 32]), hist_max=hist, kv_heads=kvh, head_dim=hd, window=window, page=page, kv=kv,
                append=rng.random() < 0.5, idle=idle, pad=rng.choice([0, 0, 3]))


def _spread(n, lo, hi):
    """n whole numbers between lo and hi, their logarithms even, in a fixed shuffled order."""
    if n == 1:
        return [hi]
    v = [min(hi, max(lo, int(round(math.exp(math.log(lo + 1) + (math.log(hi + 1) - math.log(lo + 1)) * i / (n - 1))) - 1)))
         for i in range(n)]
    step = next(k for k in (7, 5, 3, 11, 13, 1) if math.gcd(k, n) == 1)
    return [v[i * step % n] for i in range(n)]


def _lens(case):
    """(tokens of the tree, keys) of each sequence; an idle batch has every fifth one empty."""
    n = case["seqs"]
    new = _spread(n, case["tree_min"], case["tree_max"])
    keys = [a + b for a, b in zip(new, _spread(n, case["hist_min"], case["hist_max"])[::-1])]
    if case["idle"]:
        for i in range(1, n, 5):
            new[i] = keys[i] = 0
    return new, keys


def _type(name):
    return torch.float16 if name == "f16" else torch.float32


def _on(x, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV).to(dtype)


def _parents(new, r):
    """Parents of packed trees: node 0 is the sequence's last sure token, the others hang from earlier ones, later
    ones deeper (about log n levels); now and then a second root."""
    out = []
    for n in new:
        i = np.arange(n)
        p = np.floor(i * r.random(n) ** 0.6).astype(np.int64)
        p = np.where(r.random(n) < 0.02, -1, p)
        if n:
            p[0] = -1
        out.append(p)
    return np.concatenate(out) if out else np.zeros(0, np.int64)


def _pages(counts, r, spare, lows=None):
    """A table of counts[b] pages each from a shuffled pool, those in front of lows[b] given back, and the pool's size."""
    cols = max(1, max(counts)) + 1
    lows = lows or [0] * len(counts)
    table = np.full((len(counts), cols), -1, np.int64)
    used = 0
    for b, c in enumerate(counts):
        lo = min(lows[b], c)
        table[b, lo:c] = np.arange(used, used + c - lo)
        used += c - lo
    perm = r.permutation(used + spare)
    return np.where(table >= 0, perm[np.maximum(table, 0)], -1), used + spare, perm[used:]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    r = np.random.default_rng(int(seed))

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    kind = case["kind"]
    s = dict(kind=kind)
    if kind == "beam":
        B, W, V = case["groups"], case["beams"], case["vocab"]
        x = 3 * randn(B * W, V)
        x += 0.5 * x.abs().pow(1.5).copysign(x)  # a long upper tail: a few likely tokens
        s.update(groups=B, beams=W, vocab=V, out=case["out"], cap=case["cap"], logits=x.to(_type(case["logits"])))
        s["scores"] = -5 - 3 * torch.rand(B, W, device=DEV, generator=g)
        if case["first"]:  # the first step: all beams are the prompt's copies, one counts
            s["scores"][:, 1:] = float("-inf")
        s["done"] = (torch.rand(B, W, device=DEV, generator=g) < 0.2) if case["done"] else None
        s["pad"] = 1
    elif kind == "fork":
        B, W, page = case["groups"], case["beams"], case["page"]
        prompt, grown = _spread(B, case["prompt_min"], case["prompt_max"]), _spread(B, case["grown_min"], case["grown_max"])
        keys = np.array([[a + b] * W for a, b in zip(prompt, grown)]).reshape(-1)
        shared = np.array([[a // page] * W for a in prompt]).reshape(-1)  # a prompt's full pages are its beams' common ones
        cols = int(keys.max() + case["room"] + page - 1) // page + 1
        table, used = np.full((B * W, cols), -1, np.int64), 0
        for j in range(B * W):
            n = -(-int(keys[j]) // page)
            first = int(shared[j])
            if j % W == 0:
                table[j, :first] = np.arange(used, used + first)
                used += first
            table[j, :first] = table[j - j % W, :first]
            table[j, first:n] = np.arange(used, used + n - first)
            used += n - first
        n_pages = used + B * W * (2 + case["room"] // page) + 3
        perm = r.permutation(n_pages)
        s.update(room=case["room"], page=page, n_pages=n_pages, table=_on(np.where(table >= 0, perm[np.maximum(table, 0)], -1)),
                 key_len=_on(keys), parent=_on(np.arange(B * W) // W * W + r.integers(0, W, B * W)), cols=cols)
        s["free"] = _on(np.concatenate([perm[used:], np.full(used, -1)]))
        s["n_free"] = _on(np.array([n_pages - used]))
    else:
        new, keys = _lens(case)
        cu = np.concatenate([[0], np.cumsum(new)])
        tokens = int(cu[-1])
        rows = max(1, tokens + case["pad"])  # rows behind the last sequence belong to nobody
        par = np.concatenate([_parents(new, r), np.full(rows - tokens, -1)])
        s.update(seqs=case["seqs"], tokens=tokens, n_max=max(1, max(new)), t_max=max(1, max(keys)), cu=_on(cu), key_len=_on(keys),
                 parents=_on(par))
        if kind != "tree":
            # drafts that the model agrees with two times in three
            t = np.concatenate([np.repeat(cu[:-1], new), np.zeros(rows - tokens, np.int64)]) + np.maximum(par, 0)
            targets = r.integers(0, 40, rows)
            s["targets"] = _on(targets)
            s["drafts"] = _on(np.where(r.random(rows) < 0.67, targets[t], r.integers(0, 40, rows)))
            s["max_path"] = min(s["n_max"], 64)
        if kind != "accept":
            page, w = case["page"], case.get("window", 0)
            lows = [max(0, k - n + 1 - w) // page if w else 0 for n, k in zip(new, keys)]
            table, s["n_pages"], _ = _pages([-(-k // page) for k in keys], r, 3, lows)
            s.update(page=page, table=_on(table), hd=case["head_dim"], kvh=case["kv_heads"], window=w)
        if kind == "tree":
            hd, kvh, kv = s["hd"], s["kvh"], _type(case["kv"])
            s["k_pages"] = (GAIN * randn(s["n_pages"], page, kvh, hd)).to(kv)
            s["v_pages"] = randn(s["n_pages"], page, kvh, hd).to(kv)
            s["q_gain"], s["k_gain"] = GAIN * (1 + 0.1 * randn(hd)), GAIN * (1 + 0.1 * randn(hd))
            # RoPE tables by absolute position, made in 64 bits: 1e4 at sliding layers, 1e6 at global ones
            inv = (1e4 if w else 1e6) ** (-torch.arange(hd // 2, dtype=torch.float64, device=DEV) / (hd // 2))
            ang = torch.arange(s["t_max"], dtype=torch.float64, device=DEV)[:, None] * inv
            s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
            s["q"], s["append"] = randn(rows, NH, hd), case["append"]
            s["out"] = torch.zeros(rows, NH, hd, dtype=torch.float16, device=DEV)
            if s["append"]:
                s["k_new"], s["v_new"] = randn(rows, kvh, hd), randn(rows, kvh, hd)
        elif kind == "keep":
            s["path"], s["n_path"], _, _ = _accept(s)
    if kind in ("keep", "fork"):
        shape = (s["n_pages"], case["page"], case["kv_heads"], case["head_dim"])
        s["pools"] = [randn(*shape).to(_type(case["kv"])) for _ in range(2 * case["layers"])]
    if own:
        import slang_amd as sa
        s["ws"] = sa.Workspace()
        if kind == "tree":
            s["cfg"] = sa.AttnConfig(NH, s["kvh"], s["hd"], s["window"])
    return s


# ---------------------------------------------------------------- the plain forms
def _rows(s):
    """Of each packed row: its sequence and its index in the tree; the parents [seqs][n] of a padded batch, -1 a root."""
    cu = s["cu"].long()
    tok = torch.arange(s["tokens"], device=DEV)
    b = torch.searchsorted(cu[1:], tok, right=True)
    i = tok - cu[b]
    par = torch.full((s["seqs"], s["n_max"]), -1, dtype=torch.long, device=DEV)
    par[b, i] = s["parents"][:s["tokens"]].long()
    at = torch.arange(s["n_max"], device=DEV)
    return b, i, torch.where((par >= 0) & (par < at), par, -1)


def _ancestors(par):
    """[seqs][n][n]: 1 where j is i or one of its ancestors, by squaring the relation of one step."""
    n = par.shape[1]
    a = torch.eye(n, device=DEV).expand(par.shape[0], n, n).clone()
    a += (par[..., None] == torch.arange(n, device=DEV)).float()
    for _ in range(max(1, (n - 1).bit_length())):
        a = (torch.matmul(a, a) > 0).float()
    return a


def _accept(s):
    """path [seqs][max_path] (-1 behind its end), its length, the token that the model adds to it, the keys that stay."""
    b, i, par = _rows(s)
    n, P = s["n_max"], s["max_path"]
    there = torch.zeros(s["seqs"], n, dtype=torch.bool, device=DEV)
    there[b, i] = True
    draft, target = (torch.full((s["seqs"], n), -1, dtype=torch.long, device=DEV) for _ in range(2))
    draft[b, i], target[b, i] = s["drafts"][:s["tokens"]].long(), s["targets"][:s["tokens"]].long()
    ok = there & (par >= 0) & (draft == target.gather(1, par.clamp(min=0)))
    at = torch.arange(n, device=DEV)
    # only the first of the children that match
    first = torch.full((s["seqs"], n + 1), n, dtype=torch.long, device=DEV)
    first.scatter_reduce_(1, torch.where(ok, par, n), at.expand_as(par), "amin")
    ok &= first.gather(1, par.clamp(min=0)) == at
    ok[:, 0] = there[:, 0]
    taken = torch.matmul(_ancestors(par), (~ok).float()[..., None])[..., 0] == 0
    rank = taken.cumsum(1) - 1
    taken &= rank < P
    path = torch.full((s["seqs"], P + 1), -1, dtype=torch.long, device=DEV)
    path.scatter_(1, torch.where(taken, rank, P), at.expand_as(par).contiguous())
    path = path[:, :P].contiguous()
    count = taken.sum(1)
    path[torch.arange(P, device=DEV) >= count[:, None]] = -1
    last = path.gather(1, (count - 1).clamp(min=0)[:, None])
    nxt = torch.where(count > 0, target.gather(1, last.clamp(min=0))[:, 0], -1)
    cu = s["cu"].long()
    kept = s["key_len"].long() - (cu[1:] - cu[:-1]) + count
    return path.int(), count.int(), nxt.int(), kept.int()


def _rms(x):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)


def _rot(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _tree(s):
    b, i, par = _rows(s)
    anc = _ancestors(par)
    depth = anc.sum(-1).long() - 1
    n, N, T, kvh, hd, G = s["seqs"], s["n_max"], s["t_max"], s["kvh"], s["hd"], NH // s["kvh"]
    cu = s["cu"].long()
    hist = s["key_len"].long() - (cu[1:] - cu[:-1])
    pos = hist[:, None] + depth
    cos, sin = s["cos"][pos[b, i]][:, None], s["sin"][pos[b, i]][:, None]
    if s["append"]:
        row = hist[b] + i
        at = s["table"][b, row // s["page"]].long() * s["page"] + row % s["page"]
        s["k_pages"].view(-1, kvh, hd)[at] = _rot(_rms(s["k_new"][:s["tokens"]]) * s["k_gain"], cos, sin).to(s["k_pages"].dtype)
        s["v_pages"].view(-1, kvh, hd)[at] = _rms(s["v_new"][:s["tokens"]]).to(s["v_pages"].dtype)
    q = torch.zeros(n, N, NH, hd, device=DEV)
    q[b, i] = _rot(_rms(s["q"][:s["tokens"]]) * s["q_gain"], cos, sin)
    t = torch.arange(T, device=DEV)
    seen = (t < hist[:, None, None]).expand(n, N, T).clone()
    if s["window"]:
        seen &= t > pos[..., None] - s["window"]
        anc = anc * ((depth[:, :, None] - depth[:, None, :]) < s["window"])
    j = t - hist[:, None]  # the key's index in the tree
    tree = anc.gather(2, j.clamp(0, N - 1)[:, None].expand(n, N, T)) > 0
    seen |= tree & ((j >= 0) & (t < s["key_len"][:, None]))[:, None]
    idx = s["table"][:, :-(-T // s["page"])].clamp(min=0).long()
    k = s["k_pages"][idx].flatten(1, 2)[:, :T].float()  # [n][T][kvH][hd]
    v = s["v_pages"][idx].flatten(1, 2)[:, :T].float()
    q = q.view(n, N, kvh, G, hd).permute(0, 2, 3, 1, 4).reshape(n, kvh, G * N, hd)
    sc = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(n, kvh, G, N, T)
    sc.masked_fill_(~seen[:, None, None], float("-inf"))
    p = torch.exp_(sc.sub_(sc.amax(-1, keepdim=True).clamp(min=-1e30)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, kvh, -1, T), v.permute(0, 2, 1, 3).contiguous()).view(n, kvh, G, N, hd)
    o = torch.where(total > 0, o / total.clamp(min=1e-30), torch.zeros_like(o))
    s["out"][:s["tokens"]] = o.permute(0, 3, 1, 2, 4).reshape(n, N, NH, hd)[b, i].half()
    return (s["out"], s["k_pages"], s["v_pages"]) if s["append"] else s["out"]


def _keep(s):
    cu, page = s["cu"].long(), s["page"]
    hist = s["key_len"].long() - (cu[1:] - cu[:-1])
    b, d = ((torch.arange(s["path"].shape[1], device=DEV) < s["n_path"][:, None]).nonzero(as_tuple=True))
    at = [s["table"][b, row // page].long() * page + row % page for row in (hist[b] + s["path"][b, d].long(), hist[b] + d)]
    for pool in s["pools"]:
        rows = pool.view(-1, *pool.shape[2:])
        rows[at[1]] = rows[at[0]]
    return s["pools"]


def _beam(s):
    B, W, V, k = s["groups"], s["beams"], s["vocab"], s["out"]
    x = s["logits"].double()
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    m = x.amax(-1, keepdim=True)
    x -= m + (x - m).exp().sum(-1, keepdim=True).log()
    x = x.view(B, W, V) + s["scores"].double()[..., None]
    if s["done"] is not None:  # a finished beam has one candidate, itself
        x[s["done"]] = float("-inf")
        x[..., s["pad"]] = torch.where(s["done"], s["scores"].double(), x[..., s["pad"]])
    x = x.view(B, W * V)
    least = torch.topk(x, k, -1).values[:, -1:]
    tied = x == least  # of equal ones the lowest index
    pick = (x > least) | (tied & (tied.cumsum(-1) <= k - (x > least).sum(-1, keepdim=True)))
    at = pick.nonzero(as_tuple=True)[1].view(B, k)
    score, order = x.gather(1, at).sort(dim=-1, descending=True, stable=True)
    at = at.gather(1, order)
    none = score == float("-inf")
    parent = torch.arange(B, device=DEV)[:, None] * W + at // V
    return score.float(), torch.where(none, -1, parent).int(), torch.where(none, -1, at % V).int()


def _fork(s):
    page, room, n_pages, cols = s["page"], s["room"], s["n_pages"], s["cols"]
    parent = s["parent"].long()
    old, L = s["table"].long(), s["key_len"].long()[parent][:, None]
    new, c = old[parent], torch.arange(cols, device=DEV)
    n = new.shape[0]
    there = (new >= 0) & (new < n_pages)
    full = c < L // page
    mine = ~full & (c < (L + room + page - 1) // page)  # columns that the row itself will write to
    at = torch.where(there, new, n_pages)
    shared = torch.zeros(n_pages + 1, dtype=torch.bool, device=DEV)
    shared[at[full]] = True
    owner = torch.full((n_pages + 1,), n, dtype=torch.long, device=DEV)
    j = torch.arange(n, device=DEV)[:, None].expand(n, cols)
    owner.scatter_reduce_(0, at[mine], j[mine], "amin")
    keeps = mine & there & ~shared[at] & (owner[at] == j)
    tail = mine & (c * page < L)
    needs = mine & ~keeps & (there | ~tail)
    held = torch.zeros(n_pages + 1, dtype=torch.bool, device=DEV)
    held[at[full | keeps]] = True
    was = torch.zeros(n_pages + 1, dtype=torch.bool, device=DEV)
    was[torch.where((old >= 0) & (old < n_pages), old, n_pages)] = True
    freed = (was & ~held)[:n_pages].nonzero()[:, 0]  # pages that no row holds any more, in order
    free = torch.cat((s["free"][:int(s["n_free"])].long(), freed))
    jj, cc = needs.nonzero(as_tuple=True)
    got = free.flip(0)[:len(jj)]
    copied = (tail & needs)[jj, cc]
    src, dst, rows = new[jj, cc][copied], got[copied], (L[jj, 0] - cc * page)[copied]
    new = torch.where(full | keeps, new, -1)
    new[jj, cc] = got
    for pool in s["pools"]:  # rows of a page that the parent filled
        some = torch.arange(page, device=DEV) < rows[:, None]
        pool[dst] = torch.where(some[..., None, None], pool[src], pool[dst])
    left = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
    left[:len(free) - len(jj)] = free[:len(free) - len(jj)].int()
    return new.int(), L[:, 0].int(), left, torch.tensor([len(free) - len(jj)], dtype=torch.int32, device=DEV), s["pools"]


def run(s):
    kind = s["kind"]
    if not own:
        return dict(tree=_tree, accept=_accept, keep=_keep, beam=_beam, fork=_fork)[kind](s)
    import slang_amd as sa
    if kind == "tree":
        new = dict(k_new=s["k_new"], v_new=s["v_new"], k_gain=s["k_gain"]) if s["append"] else {}
        out = sa.paged_tree(s["q"], s["k_pages"], s["v_pages"], s["table"], s["key_len"], s["cu"], s["parents"], s["cfg"],
                            workspace=s["ws"], q_gain=s["q_gain"], rope_cos=s["cos"], rope_sin=s["sin"], out=s["out"],
                            max_key_len=s["t_max"], **new)
        return (out, s["k_pages"], s["v_pages"]) if s["append"] else out
    if kind == "accept":
        return sa.tree_accept(s["drafts"], s["targets"], s["parents"], s["cu"], s["key_len"], max_path=s["max_path"])
    if kind == "keep":
        sa.paged_keep(s["pools"], s["table"], s["key_len"], s["cu"], s["path"], s["n_path"], max_key_len=s["t_max"])
        return s["pools"]
    if kind == "beam":
        return sa.beam_select(s["logits"], s["scores"], cap=s["cap"], n_out=s["out"], done=s["done"], pad=s["pad"], workspace=s["ws"])
    return (*sa.paged_fork(s["pools"], s["table"], s["key_len"], s["parent"], s["free"], s["n_free"], room=s["room"],
                           workspace=s["ws"]), s["pools"])


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "beam":
        n = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": n * (4 if case["logits"] == "f32" else 2) + case["groups"] * (case["beams"] * 4 + case["out"] * 12), "flops": 4 * n}
    esz = 2 if case.get("kv") == "f16" else 4
    if kind == "fork":
        W, page = case["beams"], case["page"]
        keys = [a + b for a, b in zip(_spread(case["groups"], case["prompt_min"], case["prompt_max"]),
                                      _spread(case["groups"], case["grown_min"], case["grown_max"]))]
        cols = (max(keys) + case["room"] + page - 1) // page + 1
        # of W beams whose parents are drawn evenly about 1 in e follows a parent that another one follows already
        moved = sum(k % page for k in keys) * W / math.e if W > 1 else 0.0
        row = case["kv_heads"] * case["head_dim"] * esz
        return {"bytes": case["groups"] * W * cols * 8 + 2 * moved * row * 2 * case["layers"], "flops": 0}
    new, keys = _lens(case)
    if kind == "accept":
        return {"bytes": 12 * sum(new) + 16 * case["seqs"], "flops": 0}
    row = case["kv_heads"] * case["head_dim"]
    if kind == "keep":  # paths of about two drafts beside the root, most of them not in place
        return {"bytes": 16 * case["seqs"] + sum(2 for n in new if n > 2) * 2 * row * esz * 2 * case["layers"], "flops": 0}
    hd, w, total, pairs = case["head_dim"], case["window"], 0, 0
    for n, k in zip(new, keys):
        hist = k - n
        first = max(0, hist + 1 - w) if w else 0
        total += (k - first) * row * 2 * esz  # each attended row once
        pairs += n * (hist - first + 1 + (0.6 * math.log(n) if n else 0))
    total += sum(new) * (NH * hd * (4 + 2) + 4 + (row * 2 * 4 if case["append"] else 0))
    return {"bytes": total, "flops": 4 * pairs * NH * hd}


# ---------------------------------------------------------------- the definition, in 64 bits, token by token
def _walk(parents, i):
    """The token i and its ancestors, nearest first."""
    line = [i]
    while 0 <= parents[line[-1]] < line[-1]:
        line.append(int(parents[line[-1]]))
    return line


def _paths(s):
    """Each sequence's accepted path."""
    cu, par, drafts, targets = (s[k].cpu().numpy() for k in ("cu", "parents", "drafts", "targets"))
    found = []
    for b in range(s["seqs"]):
        p, d, t = (x[cu[b]:cu[b + 1]] for x in (par, drafts, targets))
        path = [0] if len(p) else []
        while path and len(path) < s["max_path"]:
            child = [c for c in range(path[-1] + 1, len(p)) if p[c] == path[-1] and d[c] == t[path[-1]]]
            if not child:
                break
            path.append(child[0])
        found.append((path, t))
    return found


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "beam":
        W, V = s["beams"], s["vocab"]
        score, parent, token = [], [], []
        for b in range(s["groups"]):
            cand = []
            for w in range(W):
                at = float(s["scores"][b, w].double())
                if at == float("-inf"):
                    continue
                if s["done"] is not None and bool(s["done"][b, w]):
                    cand.append((-at, w, s["pad"]))
                    continue
                x = s["logits"][b * W + w].double()
                x = s["cap"] * torch.tanh(x / s["cap"]) if s["cap"] else x
                lp = x - torch.logsumexp(x, 0) + at
                vals, order = torch.sort(lp, descending=True, stable=True)
                cand += [(-v, w, t) for v, t in zip(vals[:s["out"]].tolist(), order[:s["out"]].tolist())]
            cand = sorted(cand)[:s["out"]]
            cand += [(float("inf"), None, None)] * (s["out"] - len(cand))
            score.append([-c[0] for c in cand])
            parent.append([-1 if c[1] is None else b * W + c[1] for c in cand])
            token.append([-1 if c[1] is None else c[2] for c in cand])
        return torch.tensor(score, dtype=torch.float64), torch.tensor(parent, dtype=torch.int32), torch.tensor(token, dtype=torch.int32)
    if kind == "fork":
        table, keys, parent, free = (s[k].cpu().tolist() for k in ("table", "key_len", "parent", "free"))
        page, room = s["page"], s["room"]
        free = free[:int(s["n_free"])]
        n = len(parent)
        new = [[-1] * s["cols"] for _ in range(n)]
        length = [keys[p] for p in parent]
        shared, todo = set(), []
        for j in range(n):
            for c in range(length[j] // page):
                new[j][c] = table[parent[j]][c]
                shared.add(new[j][c])
        owned = set()
        for j in range(n):
            for c in range(length[j] // page, -(-(length[j] + room) // page)):
                p = table[parent[j]][c]
                if p >= 0 and p not in shared and p not in owned:
                    owned.add(p)
                    new[j][c] = p
                elif p >= 0 or c * page >= length[j]:
                    todo.append((j, c, p))
        free += sorted({p for row in table for p in row if p >= 0} - shared - owned)
        pools = [p.clone() for p in s["pools"]]
        for j, c, p in todo:
            new[j][c] = free.pop()
            fill = length[j] - c * page
            if fill > 0:
                for x in pools:
                    x[new[j][c], :fill] = x[p, :fill]
        left = free + [-1] * (s["n_pages"] - len(free))
        i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
        return i32(new), i32(length), i32(left), i32([len(free)]), pools
    if kind == "accept":
        cu, keys = s["cu"].cpu().numpy(), s["key_len"].cpu().numpy()
        got = _paths(s)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
        return (i32([p + [-1] * (s["max_path"] - len(p)) for p, _ in got]), i32([len(p) for p, _ in got]),
                i32([int(t[p[-1]]) if p else -1 for p, t in got]),
                i32([int(keys[b] - (cu[b + 1] - cu[b]) + len(p)) for b, (p, _) in enumerate(got)]))
    cu, keys, table, page = s["cu"].cpu().numpy(), s["key_len"].cpu().numpy(), s["table"].cpu().numpy(), s["page"]
    if kind == "keep":
        src, dst = [], []
        for b, (path, _) in enumerate(_paths(s)):
            h = int(keys[b] - (cu[b + 1] - cu[b]))
            for d, i in enumerate(path):
                src.append(int(table[b, (h + i) // page]) * page + (h + i) % page)
                dst.append(int(table[b, (h + d) // page]) * page + (h + d) % page)
        for x in s["pools"]:
            flat = x.view(-1, *x.shape[2:])
            flat[dst] = flat[src].clone()
        return s["pools"]
    # the tree's attention
    f8, hd, kvh, w = torch.float64, s["hd"], s["kvh"], s["window"]
    half, par = hd // 2, s["parents"].cpu().numpy()
    theta = (1e4 if w else 1e6) ** (-torch.arange(half, dtype=f8, device=DEV) / half)

    def normed(x):
        return x * (x.square().sum(-1, keepdim=True) / hd + EPS).rsqrt()

    def rotated(x, at):  # as a complex product of the pairs (i, i + hd/2), by the tables that the call is given
        ang = at[:, None].to(f8) * theta
        z = torch.complex(x[..., :half], x[..., half:]) * torch.complex(ang.cos().float().to(f8), ang.sin().float().to(f8))[:, None]
        return torch.cat((z.real, z.imag), -1)

    kp, vp = s["k_pages"].to(f8), s["v_pages"].to(f8)
    kept = (kp.clone(), vp.clone()) if s["append"] else (kp, vp)  # in 64 bits: what is stored
    out = torch.zeros(s["q"].shape, dtype=f8, device=DEV)
    for b in range(s["seqs"]):
        lo, n = int(cu[b]), int(cu[b + 1] - cu[b])
        if not n:
            continue
        h = int(keys[b]) - n
        p = np.arange(keys[b])
        rows = torch.from_numpy(np.maximum(table[b, p // page], 0).astype(np.int64) * page + p % page).to(DEV)
        lines = [_walk(par[lo:lo + n], i) for i in range(n)]
        pos = torch.tensor([h + len(x) - 1 for x in lines], device=DEV)
        if s["append"]:
            k = rotated(normed(s["k_new"][lo:lo + n].to(f8)) * s["k_gain"].to(f8), pos)
            v = normed(s["v_new"][lo:lo + n].to(f8))
            for pool, held, x in zip((kp, vp), kept, (k, v)):
                held.view(-1, kvh, hd)[rows[h:]] = x
                pool.view(-1, kvh, hd)[rows[h:]] = x.to(s["k_pages"].dtype).to(f8)  # what is attended is what the cache holds
        q = rotated(normed(s["q"][lo:lo + n].to(f8)) * s["q_gain"].to(f8), pos)
        seen = np.zeros((n, int(keys[b])), bool)
        for i, line in enumerate(lines):
            at = h + len(line) - 1
            seen[i, max(0, at + 1 - w) if w else 0:h] = True
            seen[i, [h + j for j in (line[:w] if w else line)]] = True
        hide = ~torch.from_numpy(seen).to(DEV)
        for hh in range(NH):
            sc = q[:, hh] @ kp.view(-1, kvh, hd)[rows, hh // (NH // kvh)].T.contiguous()
            sc[hide] = float("-inf")
            out[lo:lo + n, hh] = torch.softmax(sc, -1) @ vp.view(-1, kvh, hd)[rows, hh // (NH // kvh)]
    return (out, *kept) if s["append"] else out
