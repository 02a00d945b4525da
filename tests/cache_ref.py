"""The cache operators from their definitions in 64 bits, with the rounding that each output may be off by.

Bounds count roundings: u = finfo(type).eps / 2 of the tensors' type, e = 2^-24.  A score is a sum of D products in fp32: off by
ds = ((D + 4) sum |q k| scale + 2 |s|) e at most.  exp turns that into a relative error, the sums over n keys add n e, and on the tensor cores the weights
are rounded to the tensors' type for the product with V (fp16 weights below its normal range: 2^-25 absolute, relative to a row's largest).  fp32 tensors may
also pass as pieces whose products leave 2^-22 of a score's terms behind."""
import math

import torch

E = 2.0 ** -24


def visible(T, S, length, drafts, mask, b, device):
    """[T, S or S + T]: which keys each new token sees."""
    see = torch.zeros(T, S + (T if drafts else 0), dtype=torch.bool, device=device)
    see[:, : min(max(int(length[b]), 0), S)] = True
    if drafts:
        tri = torch.ones(T, T, dtype=torch.bool, device=device).tril()
        see[:, S:] = tri if mask is None else mask[b if mask.shape[0] > 1 else 0] != 0
    return see


def attend(Q, K, V, length, Kd=None, Vd=None, mask=None, scale=0.0):
    """(out, lse, bound of out, bound of lse), all float64."""
    B, Hq, T, D = Q.shape
    Hkv, S = K.shape[1], K.shape[2]
    G = Hq // Hkv
    sc = scale or 1.0 / math.sqrt(D)
    u = torch.finfo(Q.dtype).eps / 2
    dev = Q.device
    out, out_b = (torch.zeros(B, Hq, T, D, dtype=torch.float64, device=dev) for _ in range(2))
    lse, lse_b = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device=dev), torch.zeros(B, Hq, T, dtype=torch.float64, device=dev)
    for b in range(B):
        see = visible(T, S, length, Kd is not None, mask, b, dev)
        some = see.any(dim=0)
        for h in range(Hq):
            k, v = K[b, h // G], V[b, h // G]
            if Kd is not None:
                k, v = torch.cat((k, Kd[b, h // G])), torch.cat((v, Vd[b, h // G]))
            # rows that no token sees hold anything
            k, v = torch.where(some[:, None], k, 0).double(), torch.where(some[:, None], v, 0).double()
            q = Q[b, h].double()
            x = q @ k.T * sc
            # a masked key has no effect, whatever it holds: its products are left out row by row
            x = torch.where(see, x, -math.inf)
            size = torch.where(see, q.abs() @ k.abs().T * sc, 0.0)
            m = x.amax(dim=1)
            m = torch.where(m == -math.inf, 0.0, m)
            e = torch.where(see, torch.exp(x - m[:, None]), 0.0)
            l = e.sum(dim=1)
            w = e / torch.where(l == 0, 1.0, l)[:, None]
            for t in range(T):
                vt = torch.where(see[t][:, None], v, 0.0)
                out[b, h, t] = w[t] @ vt
                n = int(see[t].sum())
                ds = float(((D + 4 + (4 if Q.dtype == torch.float32 else 0)) * size[t] + 2 * torch.where(see[t], x[t], 0.0).abs()).nan_to_num(0, 0, 0).amax()) * E if n else 0.0
                rel = 2 * ds + (n + 16) * E + (u if Q.dtype != torch.float32 else 0.0)
                wa = w[t] @ vt.abs()
                out_b[b, h, t] = rel * wa + u * out[b, h, t].abs() + (n * 2.0 ** -25 * float(vt.abs().nan_to_num(0, 0, 0).amax()) if Q.dtype == torch.float16 else 0.0) + 1e-30
                lse_b[b, h, t] = ds + (n + 16) * E + 4 * E * abs(float(m[t]))
            lse[b, h] = m + torch.log(l)
            lse[b, h][l == 0] = -math.inf
            lse_b[b, h] += 4 * E * lse[b, h].abs().nan_to_num(0, 0, 0)
    return out, lse, out_b, lse_b


def count(accepted, b, T, most):
    """The accepted tokens of a sequence: the list up to its first index that names none."""
    if accepted is None:
        return list(range(min(T, most)))
    got = []
    for t in accepted[b].tolist():
        if t < 0 or t >= T or len(got) == most:
            break
        got.append(t)
    return got


def commit(K, V, length, Kd, Vd, accepted=None, weights=None, pos=None, next_pos=None):
    """In place; returns the new lengths."""
    S, T, n = K.shape[2], Kd.shape[2], length.tolist()
    new = []
    for b in range(K.shape[0]):
        at = min(max(n[b], 0), S)
        which = count(accepted, b, T, S - at)
        for i, t in enumerate(which):
            K[b, :, at + i], V[b, :, at + i] = Kd[b, :, t], Vd[b, :, t]
            if weights is not None:
                weights[b, :, at + i] = 0
            if pos is not None:
                pos[b, :, at + i] = (at if next_pos is None else int(next_pos[b])) + i
        new.append(at + len(which))
    return torch.tensor(new, dtype=torch.int32)


def weights(Q, K, length, lse, w, accepted=None, scale=0.0):
    """(new weights float64, bound)."""
    B, Hq, T, D = Q.shape
    Hkv, S = K.shape[1], K.shape[2]
    sc = scale or 1.0 / math.sqrt(D)
    w = w.double().clone()
    bound = 2 * E * w.abs()
    for b in range(B):
        n = min(max(int(length[b]), 0), S)
        which = count(accepted, b, T, n)
        for i, t in enumerate(which):
            last = n - len(which) + i
            for h in range(Hq):
                g = h // (Hq // Hkv)
                if float(lse[b, h, t]) == -math.inf:
                    continue
                k, q, ls = K[b, g, : last + 1].double(), Q[b, h, t].double(), float(lse[b, h, t])
                x = k @ q * sc
                p = torch.exp(x - ls)
                ds = ((D + 8) * (k.abs() @ q.abs()) * sc + 4 * x.abs() + 4 * abs(ls)) * E
                w[b, g, : last + 1] += p
                bound[b, g, : last + 1] += p * (2 * ds + (len(which) * Hq // Hkv + 16) * E)
    return w, bound + 2 * E * w.abs()


def evict(K, V, length, weights, keep, sink=0, recent=0, pos=None, next_pos=None, into=None):
    """Moves rows in place or into `into`; returns (kept, new lengths)."""
    B, H, S, _ = K.shape
    kept = torch.full((B, H, keep), -1, dtype=torch.int32)
    new = []
    for b in range(B):
        n = min(max(int(length[b]), 0), S)
        m = min(n, keep)
        end = n if next_pos is None else int(next_pos[b])
        for h in range(H):
            w = weights[b, h, :n].tolist()
            at = list(range(n)) if pos is None else pos[b, h, :n].tolist()
            def order(r):
                held = at[r] < sink or at[r] >= end - recent
                return (0, 0.0, r) if held else (2, 0.0, r) if math.isnan(w[r]) else (1, -w[r], r)
            stay = sorted(sorted(range(n), key=order)[:m])
            if into is None:
                inside, late = set(stay), iter([r for r in stay if r >= m])
                source = [r if r in inside else next(late) for r in range(m)]
            else:
                source = stay
            kept[b, h, :m] = torch.tensor(source, dtype=torch.int32)
            of = torch.tensor(source, dtype=torch.long, device=K.device)
            for src, dst in zip((K, V, weights, pos), (K, V, weights, pos) if into is None else into):
                if src is not None:
                    dst[b, h, :m] = src[b, h, of].clone()
        new.append(m)
    return kept, torch.tensor(new, dtype=torch.int32)


def same(a, b):
    """Equal, NaN to NaN."""
    a, b = a.cpu(), b.cpu()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(0, 1e30, -1e30), b.nan_to_num(0, 1e30, -1e30)) if a.is_floating_point() else torch.equal(a, b)


def close(got, want, bound):
    """Within the bound where the value is finite; the same infinity, or both NaN, elsewhere."""
    got = got.double()
    fine = torch.isfinite(want)
    off = (got - want).abs()
    return bool((torch.where(fine, off <= bound, True) & (fine | (got == want) | (torch.isnan(got) & torch.isnan(want)))).all()), \
        float(torch.where(fine, off / bound.clamp(min=1e-300), 0.0).nan_to_num(math.inf).amax())
