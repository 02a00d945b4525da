"""Cases of the cache operators: attention of new tokens over a cache, and what keeps that cache.

    attend    Q [B, Hq, T, D] of T new tokens over K, V [B, Hkv, S, D] with a number of valid rows per sequence, and over the new
              tokens' own keys and values (a tree of drafts by its mask, a chain) or without those (an encoder's states)
    commit    accepted drafts become rows of the cache
    weights   the attention weight that the accepted tokens gave each row, added up
    evict     the rows of least accumulated weight leave the cache, in place or into a smaller cache

`run` computes them from elementary torch operations in 32 bits, or, with `own` set, makes the package's calls.
"""
import importlib
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _attend(dtype, B, Hq, Hkv, T, lo, hi, D, drafts, layout="head"):
    """lo, hi: rows cached for the shortest and the longest sequence; drafts: "tree", "chain" or "none" (cross attention); layout:
    "token" where Q, Kd and Vd are views of a projection's output [B, T, heads, D]."""
    return {"op": "attend", "dtype": dtype, "B": B, "Hq": Hq, "Hkv": Hkv, "T": T, "lo": lo, "hi": hi, "D": D, "drafts": drafts, "layout": layout}


def _commit(dtype, B, Hkv, T, A, lo, hi, D, layout="head"):
    """A: most accepted tokens of a sequence; 0: all T of each."""
    return {"op": "commit", "dtype": dtype, "B": B, "Hkv": Hkv, "T": T, "A": A, "lo": lo, "hi": hi, "D": D, "layout": layout}


def _weights(dtype, B, Hq, Hkv, T, A, lo, hi, D, layout="head"):
    return {"op": "weights", "dtype": dtype, "B": B, "Hq": Hq, "Hkv": Hkv, "T": T, "A": A, "lo": lo, "hi": hi, "D": D, "layout": layout}


def _evict(dtype, B, Hkv, lo, hi, keep, sink, recent, D, into):
    return {"op": "evict", "dtype": dtype, "B": B, "Hkv": Hkv, "lo": lo, "hi": hi, "keep": keep, "sink": sink, "recent": recent, "D": D, "into": into}


def listed():
    cases = {
        # one user, one new token, a short conversation: latency
        "attend_one": _attend("bf16", 1, 32, 8, 1, 777, 777, 128, "chain"),
        # continuous batching: one token for each of 64 sequences of very different lengths, a fresh one among them
        "attend_batch": _attend("bf16", 64, 32, 8, 1, 0, 8192, 128, "chain", "token"),
        # speculative decoding: trees of 48 drafted tokens over long contexts
        "attend_tree": _attend("bf16", 8, 32, 8, 48, 1000, 32768, 128, "tree", "token"),
        # a small fp32 model with a head for each key head, a small tree, odd lengths
        "attend_tree_f32": _attend("f32", 2, 8, 8, 7, 1501, 2999, 64, "tree"),
        # an encoder-decoder's cross attention over padded encoder states, ragged on both sides, a decoder block of 333 tokens
        "attend_cross": _attend("f16", 8, 16, 16, 333, 100, 1500, 64, "none", "token"),
        # a prompt's chunk of 1000 tokens behind what is cached already
        "attend_prompt": _attend("bf16", 2, 32, 8, 1000, 2000, 7001, 128, "chain", "token"),
        # up to 6 of 48 drafts accepted for each of 32 sequences
        "commit_tree": _commit("bf16", 32, 8, 48, 6, 100, 8000, 128, "token"),
        # a prompt's keys and values enter an fp32 cache whole
        "commit_prompt": _commit("f32", 4, 8, 2000, 0, 0, 1000, 64, "token"),
        # the accepted tokens' weights over the caches of a decoding batch
        "weights_step": _weights("bf16", 32, 32, 8, 48, 6, 100, 8000, 128, "token"),
        # the weights that a prompt of 700 tokens gave its own rows and those before it
        "weights_prompt": _weights("f16", 2, 16, 16, 700, 0, 0, 1801, 64),
        # a decoding step's eviction: a few rows over the budget
        "evict_step": _evict("bf16", 32, 8, 3000, 4102, 4096, 4, 256, 128, False),
        # a prompt of up to 32768 rows is reduced into a cache of 2048
        "evict_prompt": _evict("bf16", 4, 8, 9001, 32768, 2048, 4, 512, 128, True),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi + 0.5))))))


MAX_BYTES, MAX_FLOPS = 1.1e9, 1.7e11   # of the largest listed cases
F32_MAX_FLOPS = 2e9                    # fp32 is for small models


def draw(rng):
    while True:
        op = rng.choice(["attend", "attend", "attend", "commit", "weights", "evict"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        Hkv = rng.choice([1, 2, 4, 8, 16])
        group = rng.choice([1, 1, 2, 4, 5, 8])
        D = rng.choice([64, 64, 80, 96, 128, 128, 192, 256])
        B = _spread(rng, 1, 64)
        hi = _spread(rng, 50, 32768)
        lo = rng.randint(0, hi)
        layout = rng.choice(["head", "token"])
        T = _spread(rng, 1, 1000)
        A = rng.choice([0, _spread(rng, 1, min(T, 16))])
        if op == "attend":
            drafts = rng.choice(["tree", "tree", "chain", "none"])
            T = min(T, 64) if drafts == "tree" else T
            c = _attend(dtype, B, Hkv * group, Hkv, T, lo, hi, D, drafts, layout)
        elif op == "commit":
            c = _commit(dtype, B, Hkv, T, A, lo, hi, D, layout)
        elif op == "weights":
            c = _weights(dtype, B, Hkv * group, Hkv, T, A, lo, hi, D, layout)
        else:
            keep = _spread(rng, 20, 4096)
            into = rng.choice([True, False])
            hi = max(hi, keep + 1) if into else keep + _spread(rng, 1, 64)
            c = _evict(dtype, B, Hkv, min(lo, hi), hi, keep, rng.choice([0, 4]), keep // rng.choice([4, 8]), D, into)
        w = work(c)
        scores = c["B"] * c.get("Hq", 0) * c.get("T", 0) * (hi + T)
        rows = c["B"] * c["Hkv"] * (hi + T)
        # the tensors and the plain form's scores have to fit, and the rows of an eviction are sorted on the host, too
        if w["bytes"] <= MAX_BYTES and w["flops"] <= (F32_MAX_FLOPS if dtype == "f32" else MAX_FLOPS) and rows * D <= 1 << 29 and scores <= 1 << 30 and \
                (op != "evict" or rows <= 2000000):
            return c


def _lengths(case):
    """Rows cached for each sequence, from lo to hi in even steps."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [hi if B == 1 else lo + (hi - lo) * b // (B - 1) for b in range(B)]


def _accepted(case):
    """Tokens accepted for each sequence: from none to A, or all."""
    return [case["T"] if case["A"] == 0 else b % (case["A"] + 1) if case["B"] > 1 else case["A"] for b in range(case["B"])]


def _drafts_of(case):
    """Real tokens among the T of each sequence: a batch of trees is padded to its largest."""
    return [case["T"] if b % 3 == 0 else max(1, case["T"] - b % 5) for b in range(case["B"])]


class _Maker:
    def __init__(self, case, seed):
        self.case, self.td = case, DTYPES[case["dtype"]]
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def tensor(self, heads, rows, token, spread=1.0):
        B, D = self.case["B"], self.case["D"]
        shape = (B, rows, heads, D) if token else (B, heads, rows, D)
        t = torch.empty(shape, dtype=self.td, device="cuda").normal_(std=spread, generator=self.gen)
        return t.transpose(1, 2) if token else t

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.gen, device="cuda")

    def order(self, values):
        """The values as an int32 tensor, in an order drawn from the seed."""
        v = torch.tensor(values, dtype=torch.int32, device="cuda")
        return v[torch.randperm(len(values), generator=self.gen, device="cuda")].contiguous()


def _some_accepted(m, T, counts, A):
    """[B, A] int32: increasing indexes of accepted tokens, -1 behind the last."""
    B = counts.numel()
    picked = m.uniform(B, T).argsort(dim=1)[:, :A].sort(dim=1).values
    return torch.where(torch.arange(A, device="cuda") < counts[:, None], picked, -1).to(torch.int32)


def prepare(case, seed):
    m = _Maker(case, seed)
    op, B, Hkv = case["op"], case["B"], case["Hkv"]
    token = case.get("layout") == "token"
    length = m.order(_lengths(case))
    s = {"case": case, "length": length}
    if op == "attend":
        T, S = case["T"], max(case["hi"], 1)
        s.update(Q=m.tensor(case["Hq"], T, token, 1.5), K=m.tensor(Hkv, S, False), V=m.tensor(Hkv, S, False), Kd=None, Vd=None, mask=None)
        if case["drafts"] != "none":
            s.update(Kd=m.tensor(Hkv, T, token), Vd=m.tensor(Hkv, T, token))
        if case["drafts"] == "tree":
            # random trees: a token has a parent among the tokens before it and sees itself and its ancestors; padded tokens see nothing
            parent = (m.uniform(B, T) * torch.arange(T, device="cuda")).long()
            see, every = torch.eye(T, device="cuda", dtype=torch.bool).repeat(B, 1, 1), torch.arange(B, device="cuda")
            for t in range(1, T):
                see[:, t] |= see[every, parent[:, t]]
            real = torch.arange(T, device="cuda") < m.order(_drafts_of(case))[:, None]
            s["mask"] = (see & real[:, :, None]).to(torch.uint8)
    elif op == "commit":
        T, A = case["T"], case["A"]
        S = case["hi"] + (A or T)
        s.update(K=m.tensor(Hkv, S, False), V=m.tensor(Hkv, S, False), Kd=m.tensor(Hkv, T, token), Vd=m.tensor(Hkv, T, token),
                 weights=m.uniform(B, Hkv, S), pos=torch.arange(S, dtype=torch.int32, device="cuda").repeat(B, Hkv, 1), next_pos=length + 5,
                 accepted=_some_accepted(m, T, m.order(_accepted(case)), A) if A else None)
    elif op == "weights":
        # the accepted tokens are the cache's last rows already
        T, A, S = case["T"], case["A"], case["hi"] + (case["A"] or case["T"])
        counts = m.order(_accepted(case))
        s.update(Q=m.tensor(case["Hq"], T, token, 1.5), K=m.tensor(Hkv, S, False), length=length + counts, weights=m.uniform(B, Hkv, S),
                 accepted=_some_accepted(m, T, counts, A) if A else None)
        # about the size that a row's logarithm of its sum has
        s["lse"] = math.log(max(case["hi"], 2)) + 1.0 + m.uniform(B, case["Hq"], T)
    else:
        S, keep = max(case["hi"], 1), case["keep"]
        w = m.uniform(B, Hkv, S)
        # a few rows draw most of the weight, many of them none to speak of: equal values among them
        s.update(K=m.tensor(Hkv, S, False), V=m.tensor(Hkv, S, False), weights=torch.where(w < 0.5, torch.zeros_like(w), w.pow(8) * 50),
                 pos=m.uniform(B, Hkv, S).argsort(dim=2).to(torch.int32), next_pos=torch.full_like(length, S), into=None)
        if case["into"]:
            room = keep + 64
            s["into"] = (torch.zeros_like(s["K"][:, :, :1]).repeat(1, 1, room, 1), torch.zeros_like(s["V"][:, :, :1]).repeat(1, 1, room, 1),
                         torch.zeros(B, Hkv, room, device="cuda"), torch.zeros(B, Hkv, room, dtype=torch.int32, device="cuda"))
    return s


def _scores(Q, K):
    """Q K^T / sqrt(D) in fp32, [B, Hkv, group * T, keys]."""
    B, Hq, T, D = Q.shape
    Hkv = K.shape[1]
    q = Q.float().reshape(B, Hkv, Hq // Hkv * T, D)
    return torch.matmul(q, K.float().transpose(2, 3)).mul_(1.0 / math.sqrt(D))


def _plain_attend(Q, K, V, length, Kd, Vd, mask):
    B, Hq, T, D = Q.shape
    Hkv, S = K.shape[1], K.shape[2]
    G = Hq // Hkv
    there = torch.arange(S, device=Q.device) < length[:, None]
    s = _scores(Q, K).masked_fill_(~there[:, None, None], -math.inf)
    v = torch.where(there[:, None, :, None], V.float(), 0.0)
    if Kd is not None:
        see = torch.ones(T, T, dtype=torch.bool, device=Q.device).tril().expand(B, T, T) if mask is None else mask.bool()
        sd = _scores(Q, Kd).masked_fill_(~see[:, None].repeat(1, 1, G, 1), -math.inf)
        s = torch.cat((s, sd), dim=3)
        v = torch.cat((v, Vd.float()), dim=2)
    top = s.amax(dim=3, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = s.sub_(top).exp_()
    total = e.sum(dim=3, keepdim=True)
    out = torch.matmul(e, v) / torch.where(total == 0, 1.0, total)
    lse = top + total.log()
    return out.reshape(B, Hq, T, D).to(Q.dtype), lse.reshape(B, Hq, T)


def _count_accepted(accepted, T):
    """How many indexes stand before the first one outside [0, T)."""
    return ((accepted >= 0) & (accepted < T)).int().cumprod(dim=1).sum(dim=1)


def _plain_commit(s):
    K, V, Kd, Vd, length = s["K"], s["V"], s["Kd"], s["Vd"], s["length"]
    B, H, S, D = K.shape
    T = Kd.shape[2]
    index = torch.arange(T, dtype=torch.int32, device=K.device).repeat(B, 1) if s["accepted"] is None else s["accepted"]
    count = torch.minimum(_count_accepted(index, T), S - length)
    i = torch.arange(index.shape[1], device=K.device)
    b, i = torch.nonzero(i < count[:, None], as_tuple=True)
    row, of = length[b].long() + i, index[b, i].long()
    K[b, :, row] = Kd[b, :, of]
    V[b, :, row] = Vd[b, :, of]
    s["weights"][b, :, row] = 0.0
    s["pos"][b, :, row] = (s["next_pos"][b] + i).int()[:, None]
    return {"K": K, "V": V, "weights": s["weights"], "pos": s["pos"], "length": length + count.int()}


def _plain_weights(s):
    Q, K, length, lse, weights = s["Q"], s["K"], s["length"], s["lse"], s["weights"]
    B, Hq, T, D = Q.shape
    Hkv, S = K.shape[1], K.shape[2]
    index = torch.arange(T, dtype=torch.int32, device=K.device).repeat(B, 1) if s["accepted"] is None else s["accepted"]
    A = index.shape[1]
    count = _count_accepted(index, T)
    of = index.clamp(0, T - 1).long()[:, None, :].expand(B, Hq, A)
    q = Q.gather(2, of[..., None].expand(B, Hq, A, D))
    p = _scores(q, K).sub_(lse.gather(2, of).reshape(B, Hkv, -1, 1)).exp_()
    i, j = torch.arange(A, device=K.device), torch.arange(S, device=K.device)
    see = (i[None, :, None] < count[:, None, None]) & (j <= (length - count)[:, None, None] + i[None, :, None])
    p = p.masked_fill_(~see[:, None].repeat(1, 1, Hq // Hkv, 1), 0.0)
    return {"weights": weights.add_(p.sum(dim=2))}


def _plain_evict(s):
    K, V, W, P, length, case = s["K"], s["V"], s["weights"], s["pos"], s["length"], s["case"]
    B, H, S, D = K.shape
    keep = case["keep"]
    row = torch.arange(S, device=K.device)
    there = row < length[:, None, None]
    held = (P < case["sink"]) | (P >= s["next_pos"][:, None, None] - case["recent"])
    rank = torch.where(there, torch.where(held, math.inf, W), -math.inf)
    best = rank.argsort(dim=2, descending=True, stable=True)
    m = length.clamp(max=keep)
    stays = torch.zeros(B, H, S, dtype=torch.bool, device=K.device).scatter_(2, best, (row < m[:, None, None]).expand(B, H, S))
    front = (row < m[:, None, None]).expand(B, H, S)
    if s["into"] is None:
        source, target = stays & ~front, front & ~stays
        kept = torch.where(front, row, -1)
        kept[target] = row.expand(B, H, S)[source]
        out = (K, V, W, P)
    else:
        out = s["into"]
        room = out[0].shape[2]
        source, target = stays, (row[:room] < m[:, None, None]).expand(B, H, room)
        kept = torch.full((B, H, room), -1, device=K.device)
        kept[target] = row.expand(B, H, S)[source]
    for_all = torch.full((B, H, max(keep - kept.shape[2], 0)), -1, device=K.device)
    kept = torch.cat((kept, for_all), dim=2)[:, :, :keep].int()
    out[0][target], out[1][target], out[2][target], out[3][target] = K[source], V[source], W[source], P[source]
    return {"K": out[0], "V": out[1], "weights": out[2], "pos": out[3], "kept": kept, "length": m}


def _lib():
    return importlib.import_module("accelerated-final-project_b200")


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        lib = _lib()
        if op == "attend":
            out, lse = lib.cache_attend(s["Q"], s["K"], s["V"], s["length"], s["Kd"], s["Vd"], mask=s["mask"], flags=lib.FLAG_ASYNC)
            return {"out": out, "lse": lse}
        if op == "commit":
            n = lib.cache_commit(s["K"], s["V"], s["length"], s["Kd"], s["Vd"], accepted=s["accepted"], weights=s["weights"], pos=s["pos"],
                                 next_pos=s["next_pos"], flags=lib.FLAG_ASYNC)
            return {"K": s["K"], "V": s["V"], "weights": s["weights"], "pos": s["pos"], "length": n}
        if op == "weights":
            return {"weights": lib.cache_weights(s["Q"], s["K"], s["length"], s["lse"], s["weights"], accepted=s["accepted"], flags=lib.FLAG_ASYNC)}
        kept, n = lib.cache_evict(s["K"], s["V"], s["length"], s["weights"], s["case"]["keep"], sink=s["case"]["sink"], recent=s["case"]["recent"],
                                  pos=s["pos"], next_pos=s["next_pos"], into=s["into"], flags=lib.FLAG_ASYNC)
        K, V, W, P = s["into"] or (s["K"], s["V"], s["weights"], s["pos"])
        return {"K": K, "V": V, "weights": W, "pos": P, "kept": kept, "length": n}
    if op == "attend":
        out, lse = _plain_attend(s["Q"], s["K"], s["V"], s["length"], s["Kd"], s["Vd"], s["mask"])
        return {"out": out, "lse": lse}
    return {"commit": _plain_commit, "weights": _plain_weights, "evict": _plain_evict}[op](s)


def work(case):
    esz = 4 if case["dtype"] == "f32" else 2
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    rows = sum(_lengths(case))
    if case["op"] == "attend":
        Hq, T = case["Hq"], case["T"]
        Td = T if case["drafts"] != "none" else 0
        pairs = T * rows + B * (T * (T + 1) // 2 if case["drafts"] == "chain" else Td * max(1, int(math.log(T) + 1)))
        return {"bytes": float(esz * D * (2 * Hkv * (rows + B * Td) + 2 * B * Hq * T) + 4 * B * Hq * T + (B * T * T if case["drafts"] == "tree" else 0)),
                "flops": 4.0 * Hq * D * pairs}
    if case["op"] == "commit":
        n = sum(_accepted(case))
        return {"bytes": float(n * Hkv * (4 * esz * D + 8) + 8 * B), "flops": 0.0}
    if case["op"] == "weights":
        Hq, counts = case["Hq"], _accepted(case)
        # the order of lengths and counts is drawn: their means stand for them
        total = rows + sum(counts)
        pairs = sum(counts) * rows / B + sum(n * (n + 1) // 2 for n in counts)
        return {"bytes": float(Hkv * total * (esz * D + 8) + sum(counts) * Hq * (esz * D + 4)), "flops": 2.0 * Hq * D * pairs}
    kept = sum(min(n, case["keep"]) for n in _lengths(case))
    over = sum(max(0, min(n - case["keep"], case["keep"])) for n in _lengths(case))
    moved = kept if case["into"] else over
    return {"bytes": float(Hkv * (8 * rows + 4 * B * case["keep"] + moved * (4 * esz * D + 8))), "flops": 0.0}


def exact(case, seed):
    s = prepare(case, seed)
    op, B, Hkv = case["op"], case["B"], case["Hkv"]
    n = s["length"].tolist()
    if op in ("attend", "weights"):
        Q, K = s["Q"], s["K"]
        Hq, T, D = Q.shape[1], Q.shape[2], Q.shape[3]
        G = Hq // Hkv
    if op == "attend":
        out, lse = torch.zeros(B, Hq, T, D, dtype=torch.float64, device="cuda"), torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device="cuda")
        for b in range(B):
            for h in range(Hq):
                k, v = K[b, h // G, : n[b]].double(), s["V"][b, h // G, : n[b]].double()
                see = torch.ones(T, n[b], dtype=torch.bool, device="cuda")
                if s["Kd"] is not None:
                    k, v = torch.cat((k, s["Kd"][b, h // G].double())), torch.cat((v, s["Vd"][b, h // G].double()))
                    d = s["mask"][b] != 0 if s["mask"] is not None else torch.arange(T, device="cuda")[:, None] >= torch.arange(T, device="cuda")
                    see = torch.cat((see, d), dim=1)
                x = Q[b, h].double() @ k.T / D ** 0.5
                x[~see] = -math.inf
                lse[b, h] = torch.logsumexp(x, dim=1)
                out[b, h] = torch.where(lse[b, h, :, None] > -math.inf, torch.exp(x - lse[b, h, :, None].clamp(min=-1e300)), 0.0) @ v
        return {"out": out, "lse": lse}
    if op == "weights":
        w = s["weights"].double()
        for b in range(B):
            which = list(range(T)) if s["accepted"] is None else [t for t in s["accepted"][b].tolist() if t >= 0]
            first = n[b] - len(which)
            if which:
                j = torch.arange(n[b], device="cuda")
                see = j <= first + torch.arange(len(which), device="cuda")[:, None]
                for h in range(Hq):
                    x = Q[b, h, which].double() @ K[b, h // G, : n[b]].double().T / D ** 0.5
                    w[b, h // G, : n[b]] += (torch.exp(x - s["lse"][b, h, which].double()[:, None]) * see).sum(dim=0)
        return {"weights": w}
    if op == "commit":
        S, T = s["K"].shape[2], s["Kd"].shape[2]
        for b in range(B):
            which = list(range(T)) if s["accepted"] is None else [t for t in s["accepted"][b].tolist() if t >= 0]
            at = slice(n[b], n[b] + len(which))
            s["K"][b, :, at], s["V"][b, :, at] = s["Kd"][b][:, which], s["Vd"][b][:, which]
            s["weights"][b, :, at] = 0
            s["pos"][b, :, at] = int(s["next_pos"][b]) + torch.arange(len(which), dtype=torch.int32, device="cuda")
            n[b] += len(which)
        return {"K": s["K"], "V": s["V"], "weights": s["weights"], "pos": s["pos"], "length": torch.tensor(n, dtype=torch.int32)}
    keep, room = case["keep"], s["K"].shape[2] if s["into"] is None else s["into"][0].shape[2]
    kept = torch.full((B, Hkv, keep), -1, dtype=torch.int32)
    weights, pos = s["weights"].cpu().numpy(), s["pos"].cpu().numpy()
    for b in range(B):
        m = min(n[b], keep)
        for h in range(Hkv):
            w, p, end = weights[b, h, : n[b]].tolist(), pos[b, h, : n[b]].tolist(), int(s["next_pos"][b])
            held = [q < case["sink"] or q >= end - case["recent"] for q in p]
            stay = sorted(sorted(range(n[b]), key=lambda r: (not held[r], 0.0 if held[r] else -w[r], r))[:m])
            if s["into"] is None:
                inside = set(stay)
                late = iter(r for r in stay if r >= m)
                kept[b, h, :m] = torch.tensor([r if r in inside else next(late) for r in range(m)], dtype=torch.int32)
            else:
                kept[b, h, :m] = torch.tensor(stay, dtype=torch.int32)
            of = kept[b, h, :m].long().cuda()
            for src, dst in zip((s["K"], s["V"], s["weights"], s["pos"]), s["into"] or (s["K"], s["V"], s["weights"], s["pos"])):
                dst[b, h, :m] = src[b, h, of].clone()
        n[b] = m
    K, V, W, P = s["into"] or (s["K"], s["V"], s["weights"], s["pos"])
    return {"K": K, "V": V, "weights": W, "pos": P, "kept": kept, "length": torch.tensor(n, dtype=torch.int32)}
