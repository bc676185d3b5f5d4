"""The operators of drafted-token verification over a bounded KV cache: what is
measured, in elementary torch operations (`own` false) and through the
framework's calls (`own` true).

  tree    attention of T drafted tokens over n_past cached rows and each
          other's rows, a token seeing the cache and the drafted tokens that
          its mask names; optionally adding each cache row's attention weight
          to a running total per KV head
  select  the rows of each KV head worth keeping: the first and last ones and,
          of the others, those with the largest totals
  move    listed rows of the K and V caches (and their totals) moved to the
          front, in place: an accepted path's rows, or the rows that select
          kept
  score   log probabilities of given tokens, the distribution's entropy and
          its most likely alternatives, from rows of logits

Layouts are the framework's: f32 throughout, caches [n_kv][max_ctx][head_dim],
queries and outputs [token][head][head_dim].
"""
import math

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # one drafted token at a short context, the smallest decoder's heads:
        # nothing but latency
        dict(name="tree_one", op="tree", heads=14, kv=2, hd=64, n_past=37, tokens=1, tree="chain", weights=False, pad=0),
        # a drafted chain of five tokens at a context of a chat turn, 4 KV heads
        dict(name="tree_chain", op="tree", heads=32, kv=4, hd=64, n_past=2045, tokens=5, tree="chain", weights=False,
             pad=0),
        # a drafted tree of 16, queries as a slice of the fused QKV rows
        dict(name="tree_16", op="tree", heads=32, kv=8, hd=128, n_past=4001, tokens=16, tree="random", weights=False,
             pad=2048),
        # a wide tree over a long document
        dict(name="tree_64_long", op="tree", heads=32, kv=8, hd=128, n_past=32683, tokens=64, tree="random",
             weights=False, pad=0),
        # decoding one token with running totals for a later eviction
        dict(name="weights_one", op="tree", heads=32, kv=8, hd=128, n_past=16383, tokens=1, tree="chain", weights=True,
             pad=0),
        # the last tokens of a prompt vote on which of its rows matter
        dict(name="weights_window", op="tree", heads=12, kv=2, hd=128, n_past=12269, tokens=31, tree="chain",
             weights=True, pad=0),
        # eviction at a small budget
        dict(name="select_short", op="select", kv=2, n=1021, keep=512, first=4, last=32),
        # eviction of half of a long context
        dict(name="select_long", op="select", kv=8, n=131072, keep=65536, first=16, last=256),
        # an accepted path of six of 64 drafted tokens
        dict(name="move_path", op="move", kv=8, hd=128, n=4001, span=64, rows=6, per_head=False, weights=False),
        # the kept half of a long context, other rows for each head
        dict(name="move_kept", op="move", kv=8, hd=128, n=0, span=32768, rows=16384, per_head=True, weights=True),
        # one token's distribution with twenty alternatives
        dict(name="score_one", op="score", rows=1, vocab=128256, top=20),
        # every position of a verified batch
        dict(name="score_rows", op="score", rows=509, vocab=151936, top=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "select", "move", "score"])
    if op == "tree":
        heads, kv, hd = rng.choice([(14, 2, 64), (12, 2, 128), (32, 4, 64), (32, 8, 128), (16, 16, 32), (24, 3, 64)])
        tokens = _log(rng, 1, 64)
        most = min(65536, 32683 * 64 * 32 * 128 // (tokens * heads * hd), 32683 * 8 * 128 // (kv * hd))
        weights = rng.random() < 0.4
        return dict(op="tree", heads=heads, kv=kv, hd=hd, n_past=_log(rng, 16, most // 2 if weights else most),
                    tokens=tokens, tree=rng.choice(["chain", "random"]), weights=weights,
                    pad=rng.choice([0, 0, 2 * kv * hd]))
    if op == "select":
        kv, n = rng.choice([2, 3, 4, 8]), _log(rng, 200, 131072)
        first, last = rng.randrange(0, 17), rng.randrange(0, 65)
        keep = rng.randrange(first + last, n + 1)
        return dict(op="select", kv=kv, n=n, keep=keep, first=first, last=last)
    if op == "move":
        kv, hd = rng.choice([(2, 64), (4, 64), (8, 128), (2, 128)])
        if rng.random() < 0.5:
            span = rng.randrange(2, 65)
            return dict(op="move", kv=kv, hd=hd, n=_log(rng, 16, 16384), span=span, rows=rng.randrange(1, min(span, 12)),
                        per_head=False, weights=rng.random() < 0.5)
        span = _log(rng, 500, 32768)
        return dict(op="move", kv=kv, hd=hd, n=0, span=span, rows=rng.randrange(span // 4, span // 2 + 1), per_head=True,
                    weights=rng.random() < 0.5)
    vocab = rng.choice([32000, 50257, 128256, 151936, rng.randrange(1000, 152000)])
    return dict(op="score", rows=_log(rng, 1, 500), vocab=vocab, top=rng.choice([0, 1, 5, 10, 20]))


# ----------------------------------------------------------------- inputs --

def _tree_mask(tokens, parents):
    """[tokens][ceil(tokens / 32)] int32 words: bit u of row t is set where
    drafted token t sees drafted token u (itself and its ancestors)."""
    words = (tokens + 31) // 32
    rows = []
    for t in range(tokens):
        bits, u = 0, t
        while u >= 0:
            bits |= 1 << u
            u = parents[u]
        rows.append([(bits >> (32 * w)) & 0xFFFFFFFF for w in range(words)])
    m = torch.tensor(rows, dtype=torch.int64)
    return torch.where(m >= 2**31, m - 2**32, m).to(torch.int32)


_handles = []


def _backend():
    """The one handle of a program."""
    if not _handles:
        import smallm_engine_b200
        _handles.append(smallm_engine_b200.CUDABackend(0))
    return _handles[0]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    if case["op"] == "tree":
        H, kv, hd, n, T = case["heads"], case["kv"], case["hd"], case["n_past"], case["tokens"]
        max_ctx = (n + T + 255) // 256 * 256
        s["max_ctx"] = max_ctx
        s["stride"] = H * hd + case["pad"]
        # scores of a standard deviation of about 2.5, a first row that draws
        # much of the weight, values of a few units
        s["q_rows"] = 2.5 * torch.randn(T, s["stride"], device=DEV, generator=g)
        s["k"] = torch.randn(kv, max_ctx, hd, device=DEV, generator=g)
        s["v"] = torch.randn(kv, max_ctx, hd, device=DEV, generator=g)
        s["k"][:, 0] *= 1.5
        s["mask"] = None
        if case["tree"] == "random":
            c = torch.Generator().manual_seed(seed)
            r = torch.rand(T, generator=c).tolist()
            s["mask"] = _tree_mask(T, [max(-1, t - 1 - int(r[t] * min(t + 1, 9))) for t in range(T)]).to(DEV)
        s["weights"] = torch.rand(kv, max_ctx, device=DEV, generator=g) if case["weights"] else None
        s["out"] = torch.empty(T, H, hd, device=DEV)
    elif case["op"] == "select":
        # totals of many decode steps: a heavy tail
        s["max_ctx"] = (case["n"] + 255) // 256 * 256
        s["weights"] = torch.exp(2.0 * torch.randn(case["kv"], s["max_ctx"], device=DEV, generator=g))
        s["rows_out"] = torch.empty(case["kv"], case["keep"], dtype=torch.int32, device=DEV)
    elif case["op"] == "move":
        kv, hd = case["kv"], case["hd"]
        s["max_ctx"] = (case["n"] + case["span"] + 255) // 256 * 256
        s["k"] = torch.randn(kv, s["max_ctx"], hd, device=DEV, generator=g)
        s["v"] = torch.randn(kv, s["max_ctx"], hd, device=DEV, generator=g)
        s["weights"] = torch.rand(kv, s["max_ctx"], device=DEV, generator=g) if case["weights"] else None
        lists = torch.rand(kv if case["per_head"] else 1, case["span"], device=DEV, generator=g).argsort(dim=1)
        s["list"] = (case["n"] + lists[:, :case["rows"]].sort(dim=1).values).to(torch.int32).contiguous()
    else:
        rows, V, top = case["rows"], case["vocab"], case["top"]
        x = 2.5 * torch.randn(rows, V, device=DEV, generator=g)
        peak = torch.randint(0, V, (rows, 4), device=DEV, generator=g)
        s["logits"] = x.scatter_add_(1, peak, 6.0 + 4.0 * torch.rand(rows, 4, device=DEV, generator=g))
        s["tokens"] = peak[:, 0].to(torch.int32).contiguous()
        s["logprob"] = torch.empty(rows, device=DEV)
        s["entropy"] = torch.empty(rows, device=DEV)
        s["top_ids"] = torch.empty(rows, top, dtype=torch.int32, device=DEV)
        s["top_logprobs"] = torch.empty(rows, top, device=DEV)
    if own:
        # the handle and the workspace that a program keeps beside its caches
        s["be"] = _backend()
        if case["op"] == "tree":
            need = s["be"].attention_tree_workspace(case["heads"], case["kv"], case["hd"], case["n_past"],
                                                    case["tokens"], case["weights"])
            s["work"] = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------------ plain forms --

def _plain_tree(s):
    H, kv, hd, n, T = s["heads"], s["kv"], s["hd"], s["n_past"], s["tokens"]
    G = H // kv
    q = s["q_rows"][:, :H * hd].reshape(T, kv, G, hd).permute(1, 2, 0, 3).reshape(kv, G * T, hd)
    k, v = s["k"][:, :n + T], s["v"][:, :n + T]
    scores = torch.matmul(q, k.transpose(1, 2)) * (1.0 / math.sqrt(hd))
    at = torch.arange(T, device=DEV)
    if s["mask"] is None:
        seen = at[None, :] <= at[:, None]
    else:
        seen = (s["mask"].gather(1, (at // 32).expand(T, T)) >> (at % 32)) & 1 != 0
    scores.view(kv, G, T, n + T)[..., n:].masked_fill_(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    total = p.sum(dim=-1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    out = torch.matmul(p, v).view(kv, G, T, hd).permute(2, 0, 1, 3).reshape(T, H, hd)
    if s["weights"] is None:
        return out
    s["weights"][:, :n + T] += p.sum(dim=1)
    return {"out": out, "weights": s["weights"]}


def _order_key(x):
    """int64 keys in the order of the f32 values (NaN below all of them), ties
    broken by the lower index: larger key, earlier place."""
    b = (x + 0.0).view(torch.int32).to(torch.int64)
    b = torch.where(b < 0, -2147483649 - b, b)
    b = torch.where(torch.isnan(x), torch.full_like(b, -(2**31)), b)
    return b * 2**31 + (2**31 - 1 - torch.arange(x.shape[-1], device=x.device))


def _plain_select(s):
    n, keep, first, last = s["n"], s["keep"], s["first"], s["last"]
    key = _order_key(s["weights"][:, first:n - last])
    best = first + key.topk(keep - first - last, dim=1).indices.sort(dim=1).values
    head = torch.arange(first, device=DEV).expand(s["kv"], first)
    tail = torch.arange(n - last, n, device=DEV).expand(s["kv"], last)
    return torch.cat([head, best, tail], dim=1).to(torch.int32)


def _plain_move(s):
    n, c = s["n"], s["rows"]
    idx = s["list"].to(torch.int64).expand(s["kv"], c)
    wide = idx[:, :, None].expand(s["kv"], c, s["hd"])
    s["k"][:, n:n + c] = s["k"].gather(1, wide)
    s["v"][:, n:n + c] = s["v"].gather(1, wide)
    if s["weights"] is not None:
        s["weights"][:, n:n + c] = s["weights"].gather(1, idx)
    return {"k": s["k"], "v": s["v"], "weights": s["weights"]}


def _plain_score(s):
    x = s["logits"]
    top = x.amax(dim=1, keepdim=True)
    low = x - top
    e = torch.exp(low)
    total = e.sum(dim=1, keepdim=True)
    lse = torch.log(total)
    entropy = lse[:, 0] - torch.where(e > 0, e * low, torch.zeros_like(e)).sum(dim=1) / total[:, 0]
    logprob = low.gather(1, s["tokens"].to(torch.int64)[:, None]) - lse
    ids = _order_key(x).topk(s["top"], dim=1).indices
    return {"logprob": logprob[:, 0], "entropy": entropy, "top_ids": ids.to(torch.int32),
            "top_logprobs": low.gather(1, ids) - lse}


# -------------------------------------------------------- framework calls --

def _own(s):
    be = s["be"]
    if s["op"] == "tree":
        w, m = s["weights"], s["mask"]
        be.attention_tree(s["q_rows"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["out"].data_ptr(),
                          s["heads"], s["kv"], s["hd"], s["max_ctx"], s["n_past"], s["tokens"], s["work"].data_ptr(),
                          s["work"].numel(), mask=None if m is None else m.data_ptr(),
                          weights=None if w is None else w.data_ptr(), q_stride=s["stride"])
        return s["out"] if w is None else {"out": s["out"], "weights": w}
    if s["op"] == "select":
        be.cache_select(s["weights"].data_ptr(), s["kv"], s["max_ctx"], s["n"], s["keep"], s["first"], s["last"],
                        s["rows_out"].data_ptr())
        return s["rows_out"]
    if s["op"] == "move":
        w = s["weights"]
        be.cache_move(s["k"].data_ptr(), s["v"].data_ptr(), s["kv"], s["hd"], s["max_ctx"], s["list"].data_ptr(),
                      s["rows"], s["n"], per_head=s["per_head"], weights=None if w is None else w.data_ptr())
        return {"k": s["k"], "v": s["v"], "weights": w}
    be.logprobs(s["logits"].data_ptr(), s["rows"], s["vocab"], s["tokens"].data_ptr(), s["logprob"].data_ptr(),
                s["entropy"].data_ptr(), s["top"], s["top_ids"].data_ptr(), s["top_logprobs"].data_ptr())
    return {"logprob": s["logprob"], "entropy": s["entropy"], "top_ids": s["top_ids"],
            "top_logprobs": s["top_logprobs"]}


def run(state):
    if own:
        return _own(state)
    return {"tree": _plain_tree, "select": _plain_select, "move": _plain_move, "score": _plain_score}[state["op"]](state)


# -------------------------------------------------------------------- work --

def work(case):
    if case["op"] == "tree":
        H, kv, hd, n, T = case["heads"], case["kv"], case["hd"], case["n_past"] + case["tokens"], case["tokens"]
        b = 2 * kv * n * hd * 4 + 2 * T * H * hd * 4 + (T * ((T + 31) // 32) * 4 if case["tree"] == "random" else 0)
        return {"bytes": b + (8 * kv * n if case["weights"] else 0), "flops": 4 * T * H * hd * n}
    if case["op"] == "select":
        # a key and a comparison for each total
        return {"bytes": 4 * case["kv"] * (case["n"] + case["keep"]), "flops": case["kv"] * case["n"]}
    if case["op"] == "move":
        rows = case["kv"] * case["rows"]
        lists = 4 * case["rows"] * (case["kv"] if case["per_head"] else 1)
        return {"bytes": rows * (4 * case["hd"] * 4 + (8 if case["weights"] else 0)) + lists, "flops": 0}
    n = case["rows"] * case["vocab"]
    return {"bytes": 4 * n + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * n}


# ------------------------------------------------------- 64-bit definition --

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tree":
        H, kv, hd, n, T = case["heads"], case["kv"], case["hd"], case["n_past"], case["tokens"]
        out = torch.zeros(T, H, hd, dtype=torch.float64, device=DEV)
        totals = None if s["weights"] is None else s["weights"].double()
        words = None if s["mask"] is None else [[w & 0xFFFFFFFF for w in row] for row in s["mask"].tolist()]
        for t in range(T):
            vis = list(range(n)) + [n + u for u in range(T)
                                    if (u <= t if words is None else (words[t][u // 32] >> (u % 32)) & 1)]
            vis = torch.tensor(vis, device=DEV)
            for g in range(kv):
                k, v = s["k"][g, vis].double(), s["v"][g, vis].double()
                hs = slice(g * (H // kv), (g + 1) * (H // kv))
                q = s["q_rows"][t, :H * hd].view(H, hd)[hs].double()
                logit = (q @ k.T) / math.sqrt(hd)
                prob = torch.exp(logit - torch.logsumexp(logit, dim=1, keepdim=True))
                out[t, hs] = prob @ v
                if totals is not None:
                    totals[g, vis] += prob.sum(dim=0)
        return out if totals is None else {"out": out, "weights": totals}
    if case["op"] == "score":
        x = s["logits"].double()
        lp = x - torch.logsumexp(x, dim=1, keepdim=True)
        rows = torch.arange(case["rows"], device=DEV)
        best = torch.sort(s["logits"], dim=1, descending=True, stable=True).indices[:, :case["top"]]
        return {"logprob": lp[rows, s["tokens"].long()], "entropy": -(lp.exp() * lp).sum(dim=1), "top_ids": None,
                "top_logprobs": lp.gather(1, best)}
    return None
