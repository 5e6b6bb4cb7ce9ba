"""The operators of generation that branches as a server runs them: drafts checked step by step against plain decoding,
beams against a search over whole sequences; captured and replayed, on two streams, at offsets past 32 bits."""
import threading

import numpy as np
import pytest
import torch

import oracle.branching as OB
import oracle.paged as OP
import slang_amd as sa
from test_gpu_branching import beams, check_select, dev, drafted, pools_of, Pages, rows
from test_gpu_tree import Trees, tree
from paged_cases import bound, check

pytestmark = pytest.mark.gpu
V, NH, PAGE = 96, 8, 16


class Toy:
    """Layers whose q, k and v depend on the token alone, and whose outputs make the logits: attention is all it computes."""

    def __init__(self, seed, shapes=((256, 2, 0), (512, 1, 0), (256, 1, 24))):
        r = np.random.default_rng(seed)
        self.layers = []
        for hd, kvh, window in shapes:
            cos, sin = sa.rope_tables(np.arange(256), hd, 1e4, device="cpu")
            self.layers.append(dict(hd=hd, kvh=kvh, window=window, cfg=sa.AttnConfig(NH, kvh, hd, window), cos=cos.numpy(), sin=sin.numpy(),
                                    q=r.standard_normal((V, NH, hd)).astype(np.float32), k=r.standard_normal((V, kvh, hd)).astype(np.float32),
                                    v=r.standard_normal((V, kvh, hd)).astype(np.float32),
                                    gain=(0.5 + 0.1 * r.standard_normal(hd)).astype(np.float32),
                                    w=(r.standard_normal((NH * hd, V)) / np.sqrt(NH * hd)).astype(np.float32)))
        for x in self.layers:
            x["d"] = {n: torch.from_numpy(x[n]).cuda() for n in ("q", "k", "v", "gain", "w", "cos", "sin")}

    def logits(self, tokens):
        """Of the last of a list of tokens, in 64 bits (cached rows in f16)."""
        out = np.zeros(V)
        for x in self.layers:
            t = np.array(tokens)
            p = np.arange(len(t))
            k = np.stack([OP.prep(x["k"][a], x["gain"], x["cos"][i], x["sin"][i]) for i, a in enumerate(t)]).astype(np.float16).astype(np.float64)
            v = OP.rms(x["v"][t].astype(np.float64), 1e-6).astype(np.float16).astype(np.float64)
            q = OP.prep(x["q"][t[-1]], x["gain"], x["cos"][len(t) - 1], x["sin"][len(t) - 1])
            keep = p >= len(t) - x["window"] if x["window"] else p >= 0
            o = np.zeros((NH, x["hd"]))
            for h in range(NH):
                kh = h // (NH // x["kvh"])
                s = k[keep, kh] @ q[h]
                w = np.exp(s - s.max())
                o[h] = (w / w.sum()) @ v[keep, kh]
            out += o.reshape(-1) @ x["w"].astype(np.float64)
        return 8 * out

    def caches(self, n_pages):
        for x in self.layers:
            x["pages"] = [torch.zeros(n_pages, PAGE, x["kvh"], x["hd"], dtype=torch.float16, device="cuda") for _ in range(2)]
        return sa.CachePools([p for x in self.layers for p in x["pages"]])

    def attend(self, call, tok):
        """Logits of packed tokens through a paged call: call(layer, q, k_pages, v_pages, new rows)."""
        out = 0
        for x in self.layers:
            d, at = x["d"], tok.long()
            o = call(x, d["q"][at].contiguous(), *x["pages"], dict(k_new=d["k"][at].contiguous(), v_new=d["v"][at].contiguous(), k_gain=d["gain"],
                                                                    q_gain=d["gain"], rope_cos=d["cos"], rope_sin=d["sin"], out_dtype=torch.float32))
            out = out + o.flatten(1) @ d["w"]
        return 8 * out


def test_drafts_give_what_plain_decoding_gives():
    """Three sequences; each step checks a tree with right and wrong drafts, keeps what the model agrees with, and goes on;
    tokens are those of greedy decoding one by one. No length or token is read on the host but to make drafts."""
    toy, r = Toy(3), np.random.default_rng(4)
    prompts = [[5, 7, 9], [1], [11] * 20]
    steps = 14
    truth = []
    for p in prompts:  # greedy, in 64 bits; the best token is far ahead of the rounding
        s = list(p)
        for _ in range(5 * steps + 2):
            x = np.sort(toy.logits(s))
            assert x[-1] - x[-2] > 0.01, "the toy's choice is too close: another seed"
            s.append(int(np.argmax(toy.logits(s))))
        truth.append(s)
    cols = 10
    pools = toy.caches(3 * cols + 2)
    table = dev(r.permutation(3 * cols).reshape(3, cols))
    ws = sa.Workspace()
    # the prompts: chains, all of them accepted
    history = [[] for _ in prompts]
    pending = [list(p) for p in prompts]
    key_len = torch.zeros(3, dtype=torch.int32, device="cuda")
    accepted = []
    for step in range(steps):
        toks, par, new = [], [], []
        for b in range(3):
            done = len(history[b])
            if step == 0:
                t, p = pending[b], list(range(-1, len(pending[b]) - 1))
            else:  # the sure token, then drafts: some that will be right, wrong ones beside and below them
                t, p = [pending[b][0]], [-1]
                line = 0
                for depth in range(int(r.integers(0, 5))):
                    right = truth[b][done + 1 + depth]
                    kids = [int(x) for x in r.integers(0, V, int(r.integers(0, 3))) if x != right]
                    at = int(r.integers(0, len(kids) + 1)) if r.random() < 0.8 else None
                    if at is not None:
                        kids.insert(at, right)
                    base = len(t)
                    t += kids
                    p += [line] * len(kids)
                    if at is None:
                        break
                    line = base + at
            toks.append(t), par.append(p), new.append(len(t))
        cu = dev(np.concatenate([[0], np.cumsum(new)]))
        tok, parents = dev(np.concatenate(toks)), dev(np.concatenate(par))
        key_len = key_len + dev(new)
        logits = toy.attend(lambda x, q, kp, vp, kw: sa.paged_tree(q, kp, vp, table, key_len, cu, parents, x["cfg"], workspace=ws, **kw), tok)
        zero = torch.zeros(len(tok), 1, device="cuda")
        targets = sa.beam_select(logits, zero, workspace=ws)[2][:, 0].contiguous()
        if step == 0:  # a prompt is sure: its drafts are taken as they are
            targets[:-1] = torch.where(tok[1:] >= 0, tok[1:], 0)
            targets[cu[1:].long() - 1] = sa.beam_select(logits[cu[1:].long() - 1].contiguous(), zero[:3].contiguous(), workspace=ws)[2][:, 0]
        path, n_path, nxt, kept = sa.tree_accept(tok, targets, parents, cu, key_len, max_path=32)
        sa.paged_keep(pools, table, key_len, cu, path, n_path)
        key_len = kept
        for b in range(3):
            history[b] += [toks[b][i] for i in path[b, :n_path[b]].tolist()]
            pending[b] = [int(nxt[b])]
            assert history[b] + pending[b] == truth[b][:len(history[b]) + 1], (step, b)
        assert key_len.tolist() == [len(h) for h in history]
        accepted += n_path.tolist() if step else []
    assert max(accepted) >= 4 and min(accepted) == 1


def search(toy, prompt, W, steps, cap, eos):
    """Beam search over whole sequences, in 64 bits: (score, tokens) of each beam."""
    live = [(0.0, list(prompt), False)]
    for _ in range(steps):
        cand = []
        for w, (s, t, done) in enumerate(live):
            if done:
                cand.append((-s, w, 0))
                continue
            x = toy.logits(t)
            x = cap * np.tanh(x / cap) if cap else x
            lp = x - x.max() - np.log(np.exp(x - x.max()).sum())
            cand += [(-(s + lp[v]), w, v) for v in range(V)]
        cand = sorted(cand)
        gaps = [b[0] - a[0] for a, b in zip(cand[:W], cand[1:W + 1])]
        assert min(gaps) > 1e-3, "two candidates are too close: another seed"
        live = [(-c[0], live[c[1]][1] + ([c[2]] if not live[c[1]][2] else []), live[c[1]][2] or c[2] == eos) for c in cand[:W]]
    return live


@pytest.mark.parametrize("cap,eos,seed", [(0.0, -1, 3), (30.0, 3, 2)])
def test_beams_give_what_a_search_over_sequences_gives(cap, eos, seed):
    """Two prompts, four beams each: selection, forked pages and one decode a step, pages drawn from and given back to one list."""
    toy, W, steps = Toy(seed), 4, 20
    prompts = [[5, 7, 9, 4, 30], [1] * 18]
    want = [search(toy, p, W, steps, cap, eos) for p in prompts]
    cols, n = 4, 2 * W
    n_pages = 64
    pools = toy.caches(n_pages)
    ws, wf = sa.Workspace(), sa.Workspace()
    # the prompts in rows 0 and W; the others are idle until the first fork
    free = list(np.random.default_rng(1).permutation(n_pages))
    table = np.full((n, cols), -1)
    lens = np.zeros(n, int)
    for g, p in enumerate(prompts):
        lens[g * W] = len(p)
        for c in range(-(-len(p) // PAGE)):
            table[g * W, c] = free.pop()
    cu = np.concatenate([[0], np.cumsum(lens)])
    tok = dev(np.concatenate(prompts))
    par = np.concatenate([np.arange(-1, len(p) - 1) for p in prompts])
    table, lens, cu = dev(table), dev(lens), dev(cu)
    logits = toy.attend(lambda x, q, kp, vp, kw: sa.paged_tree(q, kp, vp, table, lens, cu, dev(par), x["cfg"], workspace=ws, **kw), tok)
    first = [len(prompts[0]) - 1, len(prompts[0]) + len(prompts[1]) - 1]
    logits = logits[dev(np.repeat(first, W)).long()].contiguous()
    scores = torch.full((2, W), float("-inf"), device="cuda")
    scores[:, 0] = 0
    done = torch.zeros(2, W, dtype=torch.bool, device="cuda")
    free_t = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
    free_t[:len(free)] = dev(free)
    n_free = dev([len(free)])
    seqs = torch.zeros(n, 0, dtype=torch.int32, device="cuda")
    total = n_pages
    for step in range(steps):
        scores, parent, token = sa.beam_select(logits, scores, cap=cap, done=done if eos >= 0 else None, pad=0, workspace=ws)
        assert (parent >= 0).all()
        parent, token = parent.view(-1), token.view(-1)
        was = done.view(-1)[parent.long()]
        seqs = torch.cat((seqs[parent.long()], torch.where(was, -1, token)[:, None]), 1)
        done = (was | (token == eos)).view(2, W)
        table, lens, free_t, n_free = sa.paged_fork(pools, table, lens, parent, free_t, n_free, room=1, workspace=wf)
        used = table[table >= 0].unique().numel()
        assert n_free.item() + used == total, "a page was lost"
        lens = lens + 1
        logits = toy.attend(lambda x, q, kp, vp, kw: sa.paged_decode(q, kp, vp, table, lens, x["cfg"], workspace=ws, **kw), token)
    for g in range(2):
        got = [(float(scores[g, w]), [t for t in seqs[g * W + w].tolist() if t >= 0]) for w in range(W)]
        for w in range(W):
            assert got[w][1] == want[g][w][1][len(prompts[g]):], (g, w)
            # the logits' error: f16 weights and rows of three layers, 2^-11 of sums of size 8, over the steps
            assert abs(got[w][0] - want[g][w][0]) < steps * 8 * 3 * 2.0 ** -11


def test_captured_beams_and_paths():
    """beam_select, paged_fork between two sets of buffers, tree_accept and paged_keep in one graph, replayed on new inputs."""
    page, groups, W = 16, 3, 4
    sets = []
    for seed in (1, 2, 3):
        r = np.random.default_rng(seed)
        table, keys, free, n_pages = beams(groups, W, r.integers(0, 60, groups), r.integers(1, 30, groups), page, seed, spare=60)
        sets.append([table, keys, free, n_pages])
    cols, n_pages = max(s[0].shape[1] for s in sets), max(s[3] for s in sets)
    n = groups * W
    new = [7, 0, 12]
    buf = dict(table=dev(np.zeros((n, cols))), keys=dev(np.zeros(n)), free=dev(np.zeros(n_pages)), n_free=dev([0]),
               logits=torch.zeros(n, 3000, device="cuda"), scores=torch.zeros(groups, W, device="cuda"),
               drafts=dev(np.zeros(19)), targets=dev(np.zeros(19)), parents=dev(np.zeros(19)))
    cu, k3 = dev(np.concatenate([[0], np.cumsum(new)])), dev([20, 3, 15])
    pools = sa.CachePools(pools_of(Pages(n_pages, page), 2, 3))
    ws = sa.Workspace().reserve(max(sa.beam_select_ws_bytes(groups, W, 3000), sa.paged_fork_ws_bytes(n_pages, n)))
    out = [torch.zeros(groups, W, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]
    fk = [dev(np.zeros((n, cols))), dev(np.zeros(n)), dev(np.zeros(n_pages)), dev([0])]
    ac = [dev(np.zeros((3, 8))), dev(np.zeros(3)), dev(np.zeros(3)), dev(np.zeros(3))]

    def step():
        sa.beam_select(buf["logits"], buf["scores"], out=out, workspace=ws)
        sa.paged_fork(pools, buf["table"], buf["keys"], out[1].view(-1), buf["free"], buf["n_free"], out=fk, workspace=ws)
        sa.tree_accept(buf["drafts"], buf["targets"], buf["parents"], cu, k3, out=ac, max_path=8)
        sa.paged_keep(pools, fk[0][:3], k3, cu, ac[0], ac[1])

    def load(i):
        table, keys, free, pages = sets[i]
        t = np.full((n, cols), -1)
        t[:, :table.shape[1]] = table
        f = np.full(n_pages, -1)
        f[:len(free)] = free
        par, drafts, targets = drafted(new, i)
        for name, x in (("table", t), ("keys", keys), ("free", f), ("n_free", [len(free)]), ("drafts", drafts), ("targets", targets),
                        ("parents", par)):
            buf[name].copy_(dev(x))
        buf["logits"].copy_(torch.from_numpy(rows(n, 3000, i)))
        buf["scores"].copy_(-torch.rand(groups, W, generator=torch.Generator().manual_seed(i)))
        for j, p in enumerate(pools.tensors):
            p.copy_(torch.randn(p.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(100 * i + j)))

    load(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    everything = lambda: [x.clone() for x in (*out, *fk, *ac, *pools.tensors)]  # noqa: E731
    for i in (0, 1, 2, 1):
        load(i)
        step()
        want = everything()
        load(i)
        for x in (*out, *fk, *ac):
            x.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(everything(), want):
            assert torch.equal(a.view(torch.uint8) if a.dtype is torch.float16 else a, b.view(torch.uint8) if b.dtype is torch.float16 else b)


def test_two_threads_and_streams():
    """Calls of two threads, each on its own stream with its own workspaces, are those of one."""
    b = [Trees([900, 40, 300], [20, 5, 33], seed=s, kvh=k) for s, k in ((1, 1), (2, 2))]
    want = [tree(x, x.dev(), append=True).cpu() for x in b]
    x = rows(16, 5000, 1)
    best = [y.cpu() for y in sa.beam_select(torch.from_numpy(x).cuda(), torch.zeros(4, 4, device="cuda"), workspace=sa.Workspace())]
    bad = []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                w, d = sa.Workspace(), b[i].dev()
                lg, z = torch.from_numpy(x).cuda(), torch.zeros(4, 4, device="cuda")
                for _ in range(20):
                    got = tree(b[i], d, append=True, workspace=w)
                    sel = sa.beam_select(lg, z, workspace=w)
                    s.synchronize()
                    if not torch.equal(got.cpu(), want[i]) or any(not torch.equal(p.cpu(), q) for p, q in zip(sel, best)):
                        bad.append(i)
        except Exception as e:  # noqa: BLE001
            bad.append(e)
    t = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    [x.start() for x in t]
    [x.join() for x in t]
    assert not bad


def test_offsets_past_32_bits():
    """Pools of 5 GB and logits of 4.6 GB: the last pages and rows as the first ones."""
    n_pages, kvh, hd = 600000, 1, 256
    b = Trees([70, 40], [20, 12], kvh=kvh)
    used = sorted({int(p) for p in b.table.reshape(-1) if p >= 0})
    to = {p: n_pages - 1 - i for i, p in enumerate(used)}
    kp, vp = (torch.empty(n_pages, PAGE, kvh, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    for p, q in to.items():
        kp[q], vp[q] = torch.from_numpy(b.k_pages[p]).cuda(), torch.from_numpy(b.v_pages[p]).cuda()
    table = np.vectorize(lambda p: to.get(int(p), -1))(b.table)
    d = b.dev(k_pages=kp, v_pages=vp, table=dev(table))
    out, A, S = b.oracle()
    check(tree(b, d).cpu().numpy(), out, bound(out, A, S, q16=True, kv32=False, out16=True))
    path = np.array([[0, 3, 7, 8], [1, 2, 11, -1]])
    before = [x.reshape(-1, kvh, hd) for x in (b.k_pages, b.v_pages)]
    want = OB.keep([x.copy() for x in before], b.keys, b.cu, path, [4, 3], b.table, PAGE, b.n_pages)
    sa.paged_keep([kp, vp], d["table"], d["key_len"], d["cu"], dev(path), dev([4, 3]))
    for got, w in zip((kp, vp), want):
        for p, q in to.items():
            assert np.array_equal(got[q].cpu().numpy().view(np.uint8), w.reshape(-1, PAGE, kvh, hd)[p].view(np.uint8))
    # a fork's copies there
    free = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
    free[0] = 7
    tail = kp[to[int(b.table[0, 4])]].clone()
    got = sa.paged_fork([kp, vp], d["table"], d["key_len"], dev([0, 0]), free, dev([1]), workspace=sa.Workspace())
    assert got[0][1, 4].item() == int(table[1, 0]) or got[0][1, 4].item() in set(int(x) for x in table[1] if x >= 0)
    assert torch.equal(kp[got[0][1, 4].item(), :6].view(torch.int16), tail[:6].view(torch.int16))
    del kp, vp, d
    torch.cuda.empty_cache()
    big = torch.zeros(8800, 262144, dtype=torch.float16, device="cuda")
    x = rows(16, 262144, 3, np.float16)
    big[-16:] = torch.from_numpy(x).cuda()
    got = sa.beam_select(big, torch.zeros(1100, 8, device="cuda"), workspace=sa.Workspace())
    last = [y[-2:].cpu().numpy() for y in got]
    last[1] = last[1] - 8784
    check_select(x, np.zeros((2, 8), np.float32), got=last)
    assert got[2][:-2].cpu().eq(torch.arange(8, dtype=torch.int32)).all() and (got[1][0] == 0).all()
