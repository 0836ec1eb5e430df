"""The operators of a batch of continuations of one prompt, timed by themselves: the calls that a program which serves such a batch makes, and the same results from elementary torch operations.

  attention  every token of a pass over the cells of the shared prompt and the cells of its own continuation (pi_op_prefix_attention)
  mass       what every cell has been given by the soft-maxes of a pass, added up over its tokens and heads (pi_op_attention_mass)
  evict      the cells that keep their place when the cache is cut to a budget, and their rows brought to the front (pi_op_cache_choose, pi_op_cache_move)
  sample     a token for every row of logits: top-k, top-p, min-p, temperature, and a given random number (pi_op_sample)

Caches are those of pi_op_attention: float16 rows of all key / value heads, one per cell.  A pass of `tokens` continuations stands behind `prompt` cells that all of them see; the cells behind those were taken in turn, one step
of all continuations after the other, and continuation t sees its own ones: `own` of them, or down to half as many where it was begun later.  Inputs are synthetic.
"""
import math

import numpy as np
import torch

own = False


def listed():
    def att(name, heads, kv, dim, tokens, prompt, cells):
        return {"name": name, "kind": "attention", "heads": heads, "kv_heads": kv, "dim": dim, "tokens": tokens, "prompt": prompt, "own": cells}

    def smp(name, rows, vocab, top_k, top_p, min_p, temp, masked=False):
        return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "top_k": top_k, "top_p": top_p, "min_p": min_p, "temp": temp, "masked": masked}

    return [
        # one token of a small draft model behind a short prompt: latency
        att("attention, 1 token", 32, 4, 64, 1, 500, 13),
        # a handful of answers to one long question, eight query heads to a key head
        att("attention, 16 x 4000", 64, 8, 128, 16, 4000, 97),
        # every head with keys of its own: the caches are eight times as large
        att("attention, 24 x 2047, own keys", 32, 32, 128, 24, 2047, 64),
        # a batch of agents over one book
        att("attention, 64 x 32000", 64, 8, 128, 64, 32000, 128),
        # the weights of one step of a few continuations, for the bookkeeping of an eviction
        {"name": "mass, 8 x 3000", "kind": "mass", "heads": 32, "kv_heads": 32, "dim": 80, "tokens": 8, "prompt": 3000, "own": 61},
        {"name": "mass, 64 x 16000", "kind": "mass", "heads": 64, "kv_heads": 8, "dim": 128, "tokens": 64, "prompt": 16000, "own": 100},
        # a quarter of a short context given up, in the caches of 22 layers of a small model
        {"name": "evict, 1000 of 1331", "kind": "evict", "layers": 22, "kv_heads": 4, "dim": 64, "cells": 1331, "keep": 1000, "guard": 40},
        # half of a long one
        {"name": "evict, 16384 of 32768", "kind": "evict", "layers": 16, "kv_heads": 8, "dim": 128, "cells": 32768, "keep": 16384, "guard": 600},
        # a token of one sequence with the usual chain
        smp("sample, 1 x 32000", 1, 32000, 40, 0.95, 0.05, 0.8),
        # the same for a batch over a larger vocabulary, a grammar forbidding most of it
        smp("sample, 33 x 65024, masked", 33, 65024, 50, 0.9, 0.02, 0.7, True),
        # temperature and nucleus alone: thousands of candidates stay
        smp("sample, 64 x 131072, nucleus", 64, 131072, 0, 0.97, 0.0, 1.1),
        # every row its own settings
        smp("sample, 256 x 131072", 256, 131072, -1, -1.0, -1.0, -1.0),
    ]


HEADS = [(32, 4, 64), (32, 32, 128), (64, 8, 128), (128, 8, 64), (32, 32, 80), (64, 64, 64), (71, 1, 64), (24, 3, 96), (8, 2, 256), (20, 5, 40)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "mass", "evict", "sample", "sample"])
    largest = {c["kind"]: work(c) for c in listed()}            # (the last of a kind is its largest)
    while True:
        if kind in ("attention", "mass"):
            heads, kv, dim = rng.choice(HEADS)
            c = {"kind": kind, "heads": heads, "kv_heads": kv, "dim": dim, "tokens": _log(rng, 1, 200), "prompt": _log(rng, 1, 40000) - 1, "own": _log(rng, 1, 400)}
            if c["tokens"] * heads * (c["prompt"] + c["tokens"] * c["own"]) > 64 * 64 * (32000 + 64 * 128):         # (what the plain form holds)
                continue
        elif kind == "evict":
            cells = _log(rng, 2, 60000)
            c = {"kind": kind, "layers": _log(rng, 1, 40), "kv_heads": rng.choice([1, 2, 3, 4, 8, 32]), "dim": rng.choice([40, 64, 80, 96, 128]), "cells": cells, "keep": rng.randint(1, cells), "guard": rng.randint(0, cells // 4)}
            if c["layers"] * c["kv_heads"] * c["dim"] * cells > 16 * 8 * 128 * 32768:
                continue
        else:
            c = {"kind": kind, "rows": _log(rng, 1, 300), "vocab": _log(rng, 300, 260000), "top_k": rng.choice([0, 1, 20, 100, 1000, 40, -1]), "top_p": rng.choice([1.0, 0.95, 0.8, 0.5, -1.0]),
                 "min_p": rng.choice([0.0, 0.0, 0.05, 0.2, -1.0]), "temp": rng.choice([0.6, 1.0, 1.5, -1.0]), "masked": rng.random() < 0.25}
            if c["rows"] * c["vocab"] > 256 * 131072:
                continue
        w = work(c)
        if w["bytes"] <= largest[kind]["bytes"] and w["flops"] <= largest[kind]["flops"]:
            return c


def _cells(c):
    return c["prompt"] + c["tokens"] * c["own"]


def _lengths(c):
    """cells of its own that each continuation sees"""
    return [c["own"] - (t * 7919 % (c["own"] // 2 + 1)) for t in range(c["tokens"])]


def work(case):
    c = case
    if c["kind"] in ("attention", "mass"):
        rows, seen = c["tokens"] * c["heads"], sum(_lengths(c))
        pairs = c["heads"] * (c["tokens"] * c["prompt"] + seen)                                       # (query, cell) pairs, all heads
        cache = 2 * c["kv_heads"] * c["dim"] * (c["prompt"] + seen)                                   # one cache's rows that anybody sees
        mask = c["tokens"] * ((_cells(c) + 31) // 32 - c["prompt"] // 32) * 4
        q = 2 * rows * c["dim"]
        if c["kind"] == "attention":
            return {"bytes": q + 2 * cache + mask + 4 * rows * (c["dim"] + 1), "flops": 4 * pairs * c["dim"]}
        return {"bytes": q + cache + mask + 4 * rows + 8 * _cells(c), "flops": 2 * pairs * c["dim"]}
    if c["kind"] == "evict":
        moves = c["keep"] * (c["cells"] - c["keep"]) / c["cells"]                                     # the mean of a choice that knows nothing of places
        row = 2 * c["layers"] * 2 * c["kv_heads"] * c["dim"] + 4
        return {"bytes": c["cells"] * 4 + (c["cells"] + 31) // 32 * 4 + 4 * c["keep"] + 2 * moves * row, "flops": c["cells"]}
    return {"bytes": c["rows"] * (4 * c["vocab"] + 8 * 4), "flops": c["rows"] * c["vocab"]}


def _words(bits):
    """rows of truth values as bitmaps, 32 to a word"""
    t, n = bits.shape
    w = torch.zeros(t, (n + 31) // 32 * 32, dtype=torch.int64, device=bits.device)
    w[:, :n] = bits
    w = (w.view(t, -1, 32) << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32).contiguous()


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    s = {"case": c}
    if c["kind"] in ("attention", "mass"):
        n, T, H, KH, D = _cells(c), c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        s["q"] = (2.0 * randn(T, H, D)).half()                                                       # (scores of a standard deviation of two: some cells are heard, most are not)
        s["k"], s["v"] = randn(n, KH, D).half(), randn(n, KH, D).half()
        cell = torch.arange(n, device=dev) - c["prompt"]
        length = torch.tensor(_lengths(c), device=dev)
        t = torch.arange(T, device=dev)[:, None]
        s["seen"] = (cell[None, :] < 0) | ((cell[None, :] % T == t) & (cell[None, :] // T < length[:, None]))
        s["mask"], s["scale"], s["n"] = _words(s["seen"]), 1.0 / math.sqrt(D), n
        s["out"], s["lse"] = torch.zeros(T, H, D, device=dev), torch.zeros(T, H, device=dev)
        if c["kind"] == "mass":                                                                       # what the attention of the pass left, and what the passes before it gave
            s["lse"] = torch.logsumexp(_scores(s), -1).float().contiguous()
            s["mass"] = 3.0 * rand(n)
    elif c["kind"] == "evict":
        n = c["cells"]
        s["mass"] = rand(n) ** 4 * 50.0
        s["guarded"] = torch.zeros(n, dtype=torch.bool, device=dev)
        s["guarded"][n - min(c["guard"], c["keep"]):] = True                                          # the newest cells
        s["guard"] = _words(s["guarded"][None])
        s["k"], s["v"] = (randn(c["layers"], n, c["kv_heads"] * c["dim"]).half() for _ in range(2))
        s["pos"] = torch.arange(n, device=dev, dtype=torch.int32) + 5
        s["source"] = torch.zeros(c["keep"], dtype=torch.int32, device=dev)
    else:
        T, V = c["rows"], c["vocab"]
        x = 2.5 * randn(T, V)
        x.scatter_add_(1, torch.randint(0, V, (T, 64), generator=g, device=dev), 10.0 * rand(T, 64))   # a few tokens stand out
        if c["masked"]:
            x[rand(T, V) < 0.7] = -math.inf
        s["logits"] = x

        def setting(value, choices, dtype):
            pick = torch.tensor(choices, device=dev, dtype=dtype)[torch.randint(0, len(choices), (T,), generator=g, device=dev)]
            return pick if value < 0 else torch.full((T,), value, device=dev, dtype=dtype)

        s["temp"] = setting(c["temp"], [0.5, 0.8, 1.0, 1.3, 0.0], torch.float32)
        s["top_k"] = setting(c["top_k"], [0, 1, 10, 40, 40, 200], torch.int32)
        s["top_p"] = setting(c["top_p"], [1.0, 0.95, 0.9, 0.6], torch.float32)
        s["min_p"] = setting(c["min_p"], [0.0, 0.0, 0.05, 0.1], torch.float32)
        s["u"] = rand(T)
        s["id"], s["prob"], s["kept"] = torch.zeros(T, dtype=torch.int32, device=dev), torch.zeros(T, device=dev), torch.zeros(T, dtype=torch.int32, device=dev)
    if own:
        _hold(s)
    return s


def _hold(s):
    """what a program keeps beside its tensors: the library, the memory that an operator works in, the addresses"""
    from pipeinfer_amd import lib as L
    c, lib = s["case"], L.load()
    L.check(lib.pi_device_init(torch.cuda.current_device()), "pi_device_init")
    s["lib"], s["check"] = lib, L.check
    if c["kind"] in ("attention", "mass"):
        size = lib.pi_op_prefix_attention_scratch_floats if c["kind"] == "attention" else lib.pi_op_attention_mass_scratch_floats
        s["floats"] = size(c["dim"], c["heads"], c["kv_heads"], c["tokens"], c["prompt"], s["n"])
        s["scratch"] = torch.empty(max(1, s["floats"]), device="cuda")
    elif c["kind"] == "evict":
        import ctypes
        n = c["layers"]
        arrays = [s["k"][i].data_ptr() for i in range(n)] + [s["v"][i].data_ptr() for i in range(n)] + [s["pos"].data_ptr()]
        s["arrays"] = (ctypes.c_void_p * len(arrays))(*arrays)
        s["row_bytes"] = (ctypes.c_int64 * len(arrays))(*([2 * c["kv_heads"] * c["dim"]] * (2 * n) + [4]))
    else:
        s["bytes"] = lib.pi_op_sample_scratch_bytes(c["vocab"], c["rows"])
        s["scratch"] = torch.empty(max(1, s["bytes"]), dtype=torch.uint8, device="cuda")
    s["at"] = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}


def run(state):
    s = state
    c = s["case"]
    if own:
        return _own(s, c, s["at"], torch.cuda.current_stream().cuda_stream)
    if c["kind"] == "attention":
        return _plain_attention(s)
    if c["kind"] == "mass":
        return _plain_mass(s)
    if c["kind"] == "evict":
        return _plain_evict(s)
    return _plain_sample(s)


def _own(s, c, at, stream):
    lib, check = s["lib"], s["check"]
    if c["kind"] == "attention":
        row = c["heads"] * c["dim"]
        check(lib.pi_op_prefix_attention(at["q"], row, at["k"], at["v"], at["mask"], s["scale"], c["dim"], c["heads"], c["kv_heads"], c["tokens"], c["prompt"], s["n"], at["scratch"], s["floats"], at["out"], row, at["lse"],
                                         None, stream), "pi_op_prefix_attention")
        return {"out": s["out"], "lse": s["lse"]}
    if c["kind"] == "mass":
        check(lib.pi_op_attention_mass(at["q"], c["heads"] * c["dim"], at["k"], at["mask"], at["lse"], s["scale"], c["dim"], c["heads"], c["kv_heads"], c["tokens"], c["prompt"], s["n"], 1.0, at["scratch"], s["floats"],
                                       at["mass"], None, stream), "pi_op_attention_mass")
        return {"mass": s["mass"]}
    if c["kind"] == "evict":
        check(lib.pi_op_cache_choose(at["mass"], at["guard"], c["cells"], c["keep"], at["source"], stream), "pi_op_cache_choose")
        check(lib.pi_op_cache_move(s["arrays"], s["row_bytes"], 2 * c["layers"] + 1, at["source"], c["keep"], c["cells"], stream), "pi_op_cache_move")
        return {"source": s["source"], "k": s["k"], "v": s["v"], "pos": s["pos"]}
    check(lib.pi_op_sample(at["logits"], c["vocab"], c["vocab"], c["rows"], at["temp"], at["top_k"], at["top_p"], at["min_p"], at["u"], at["scratch"], s["bytes"], at["id"], at["prob"], at["kept"], stream), "pi_op_sample")
    return {"id": s["id"], "prob": s["prob"], "kept": s["kept"]}


def _scores(s):
    """[tokens, heads, cells]: q . k * scale, minus infinity for what a token does not see"""
    T, H, D = s["q"].shape
    KH = s["k"].shape[1]
    q = s["q"].float().view(T, KH, H // KH, D).permute(1, 0, 2, 3).reshape(KH, T * (H // KH), D).contiguous()
    k = s["k"].float().permute(1, 2, 0).contiguous()
    x = torch.bmm(q, k).view(KH, T, H // KH, -1).permute(1, 0, 2, 3).reshape(T, H, -1) * s["scale"]
    return x.masked_fill(~s["seen"][:, None, :], -math.inf)


def _plain_attention(s):
    x = _scores(s)
    T, H, n = x.shape
    KH, D = s["k"].shape[1:]
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m)
    z = p.sum(-1, keepdim=True)
    p = (p / z).view(T, KH, H // KH, n).permute(1, 0, 2, 3).reshape(KH, T * (H // KH), n).contiguous()
    v = s["v"].float().permute(1, 0, 2).contiguous()
    out = torch.bmm(p, v).view(KH, T, H // KH, D).permute(1, 0, 2, 3).reshape(T, H, D).contiguous()
    return {"out": out, "lse": (m + torch.log(z))[..., 0]}


def _plain_mass(s):
    s["mass"] += torch.exp(_scores(s) - s["lse"][..., None]).sum(1).sum(0)
    return {"mass": s["mass"]}


def _plain_evict(s):
    n, keep = s["case"]["cells"], s["case"]["keep"]
    score = torch.where(s["guarded"], math.inf, s["mass"])
    best = torch.sort(score, descending=True, stable=True)[1][:keep]
    stays = torch.zeros(n, dtype=torch.bool, device=score.device)
    stays[best] = True
    at = torch.arange(n, device=score.device)
    movers = torch.sort(torch.where(stays & (at >= keep), at, n))[0]                                  # the kept cells behind the budget, in their order; each goes to a hole in front of it
    hole = torch.cumsum((~stays[:keep]).to(torch.int64), 0) - 1
    source = torch.where(stays[:keep], at[:keep], movers[hole.clamp(min=0)])
    s["source"] = source.to(torch.int32)
    s["k"][:, :keep] = s["k"][:, source]
    s["v"][:, :keep] = s["v"][:, source]
    s["pos"][:keep] = s["pos"][source]
    return {"source": s["source"], "k": s["k"], "v": s["v"], "pos": s["pos"]}


def _plain_sample(s):
    x = s["logits"].double()
    T, V = x.shape
    x, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    rank = torch.arange(V, device=x.device)[None, :]
    d = x - x[:, :1]
    stay = (x > -math.inf) & ((s["top_k"][:, None] <= 0) | (rank < s["top_k"][:, None]))
    w = torch.exp(d) * stay
    ahead = torch.cumsum(w, -1)
    ahead = torch.cat([torch.zeros_like(ahead[:, :1]), ahead[:, :-1]], -1)
    p = s["top_p"].double()[:, None]
    stay &= (p >= 1) | (rank == 0) | (ahead < p * w.sum(-1, keepdim=True))
    stay &= (rank == 0) | (w >= s["min_p"].double()[:, None])
    temp = s["temp"].double()[:, None]
    e = torch.where(temp > 0, torch.exp(d / torch.where(temp > 0, temp, 1.0)), (rank == 0).double()) * stay
    e = torch.zeros_like(e).scatter_(1, ids, e)                                                      # in the order of the ids, as the number that is drawn goes along them
    cum = torch.cumsum(e, -1)
    total = cum[:, -1:]
    last = torch.where(e > 0, torch.arange(V, device=x.device)[None, :], 0).amax(-1)
    pick = torch.minimum((cum <= s["u"].double()[:, None] * total).sum(-1), last)
    prob = torch.gather(e, 1, pick[:, None])[:, 0] / total[:, 0]
    return {"id": pick.to(torch.int32), "prob": prob.float(), "kept": stay.sum(-1).to(torch.int32)}


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["kind"] in ("attention", "mass"):
        T, H, KH, D, P = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["prompt"]
        q, k, v = (s[n].double() for n in ("q", "k", "v"))
        per, lengths = H // KH, _lengths(c)
        out, lse = torch.zeros(T, H, D, dtype=torch.float64, device="cuda"), torch.zeros(T, H, dtype=torch.float64, device="cuda")
        mass = s["mass"].double() if c["kind"] == "mass" else None
        for t in range(T):
            cells = torch.cat([torch.arange(P, device="cuda"), P + t + T * torch.arange(lengths[t], device="cuda")])
            for j in range(KH):
                x = q[t, j * per:(j + 1) * per] @ k[cells, j].T.contiguous() / math.sqrt(D)
                if mass is not None:
                    mass.index_add_(0, cells, torch.exp(x - s["lse"][t, j * per:(j + 1) * per, None].double()).sum(0))
                    continue
                lse[t, j * per:(j + 1) * per] = torch.logsumexp(x, -1)
                out[t, j * per:(j + 1) * per] = torch.softmax(x, -1) @ v[cells, j]
        return {"mass": mass.cpu().numpy()} if mass is not None else {"out": out.cpu().numpy(), "lse": lse.cpu().numpy()}
    if c["kind"] == "evict":
        n, keep, guarded, mass = c["cells"], c["keep"], s["guarded"].cpu().numpy(), s["mass"].cpu().numpy().astype(np.float64)
        best = sorted(range(n), key=lambda i: (not guarded[i], -mass[i], i))[:keep]
        stays = set(best)
        later = iter(sorted(i for i in best if i >= keep))
        source = np.array([i if i in stays else next(later) for i in range(keep)], np.int64)
        res = {"source": source.astype(np.int32)}
        for name in ("k", "v", "pos"):
            a = s[name].cpu().numpy()
            a = a.astype(np.float64) if name != "pos" else a
            if name == "pos":
                a[:keep] = a[source]
            else:
                a[:, :keep] = a[:, source]
            res[name] = a
        return res
    x, top_k, top_p, min_p, temp, u = (s[n].cpu().numpy() for n in ("logits", "top_k", "top_p", "min_p", "temp", "u"))
    ids, probs, kept = [], [], []
    for t in range(c["rows"]):
        row = x[t].astype(np.float64)
        order = np.argsort(-row, kind="stable")
        order = order[np.isfinite(row[order])]
        if top_k[t] > 0:
            order = order[:top_k[t]]
        w = np.exp(row[order] - row[order[0]])
        if top_p[t] < 1:
            n = 1 + int(np.searchsorted(np.cumsum(w), np.float64(top_p[t]) * w.sum(), side="left"))
            order, w = order[:n], w[:n]
        if min_p[t] > 0:
            n = max(1, int((w >= np.float64(min_p[t])).sum()))
            order = order[:n]
        kept.append(len(order))
        if temp[t] <= 0:
            ids.append(order[0])
            probs.append(1.0)
            continue
        mine = np.sort(order)
        e = np.exp((row[mine] - row[order[0]]) / np.float64(temp[t]))
        cum = np.cumsum(e)
        i = min(int(np.searchsorted(cum, np.float64(u[t]) * cum[-1], side="right")), len(mine) - 1)
        ids.append(mine[i])
        probs.append(e[i] / cum[-1])
    return {"id": np.array(ids, np.int32), "prob": np.array(probs), "kept": np.array(kept, np.int32)}
