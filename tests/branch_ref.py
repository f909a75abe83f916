"""Plain definitions of the branching operators (64-bit, loops), for the tests."""
import numpy as np

PAGE = 16


def tree_attention(q, ka, va, n_layer, layer, bt, starts, ctx, seen, hkv, scale):
    """(out, tol): q [n_tok, hq, d] f32; seen[i] = set of visible drafted tokens of row i.

    tol bounds the kernel's error per output: q and p enter the products as two fp16 halves (each
    rounding half a step, 2^-11, so 2^-22 together), products are summed in fp32 whose steps may be
    truncated (2^-23 each): a score of d terms, two halves each, is off by at most
    e = (2^-22 + 2 d 2^-23) scale sum |q k|; a weight exp(s - m) then by a factor 1 +- 2 e + 2^-21 (exp
    and its argument), its halves by 2^-22, and the sums over n keys by 2 n 2^-23 of sum p |v|; the
    denominator has the same errors as the numerator, hence the factor two."""
    n_tok, hq, d = q.shape
    nrep = hq // hkv
    out = np.zeros(q.shape)
    tol = np.zeros(q.shape)
    for s in range(len(ctx)):
        a, b, n = int(starts[s]), int(starts[s + 1]), int(ctx[s])
        if a == b:
            continue
        hist = n - (b - a)
        rows = [int(bt[s, j // PAGE]) * n_layer + layer for j in range(n)]
        k = np.stack([ka[r, j % PAGE] for j, r in enumerate(rows)]).astype(np.float64)   # [n, hkv, d]
        v = np.stack([va[r, j % PAGE] for j, r in enumerate(rows)]).astype(np.float64)
        for i in range(a, b):
            at = list(range(hist)) + sorted(hist + t for t in seen[i])
            if not at:
                continue
            for h in range(hq):
                kk, vv, x = k[at, h // nrep], v[at, h // nrep], q[i, h].astype(np.float64)
                sc = kk @ x * scale
                p = np.exp(sc - sc.max())
                out[i, h] = p @ vv / p.sum()
                e = (2.0 ** -22 + 2 * d * 2.0 ** -23) * scale * (np.abs(kk) @ np.abs(x)).max()
                tol[i, h] = 2 * (2 * e + 2.0 ** -21 + 2.0 ** -22 + 2 * len(at) * 2.0 ** -23) * (p @ np.abs(vv)) / p.sum()
    return out, tol


def fork(t, refs, lens, held, parents, reserve, fill):
    """kv_fork on lists, in place of copies: returns (tables, refs, lens, held, copies, status) with
    copies = [(from, to, slots)]; on a bad input or too few blocks everything comes back as it was."""
    n, mbs, nb = len(t), len(t[0]), len(refs)
    old = ([list(r) for r in t], list(refs), list(lens), list(held))
    for i in range(n):
        p = parents[i]
        bad = not -1 <= p < n or not 0 <= held[i] <= mbs or reserve[i] < 0 and p >= 0
        if not bad:
            bad = any(not 0 <= b < nb for b in t[i][:held[i]])
            if i in parents:
                bad = bad or lens[i] < 0 or -(-lens[i] // PAGE) > held[i]
        if bad:
            return (*old, [], -1)
        if p >= 0 and 0 <= p < n and -(-(lens[p] + reserve[i]) // PAGE) > mbs:
            return (*old, [], -1)
    refs = list(refs)
    for i in range(n):
        for b in t[i][:held[i]]:
            refs[b] -= 1
    rows, ln = [], []
    for p in parents:
        ln.append(lens[p] if p >= 0 else 0)
        rows.append(list(t[p][:-(-ln[-1] // PAGE)]) if p >= 0 else [])
        for b in rows[-1]:
            refs[b] += 1
    free = [b for b in range(nb) if refs[b] == 0]
    asked, copies = 0, []

    def take():
        nonlocal asked
        asked += 1
        return free[asked - 1] if asked <= len(free) else 0

    for i, p in enumerate(parents):
        if ln[i] % PAGE and refs[rows[i][-1]] > 1:
            b = take()
            copies.append((rows[i][-1], b, ln[i] % PAGE))
            refs[rows[i][-1]] -= 1
            refs[b] = 1
            rows[i][-1] = b
        while p >= 0 and len(rows[i]) * PAGE < ln[i] + reserve[i]:
            b = take()
            refs[b] = 1
            rows[i].append(b)
    if asked > len(free):
        return (*old, [], asked - len(free))
    tables = [r + [fill if j < held[i] else t[i][j] for j in range(len(r), mbs)] for i, r in enumerate(rows)]
    return tables, refs, ln, [len(r) for r in rows], copies, 0


def beam(x, scores, n_beams, k, finished=None, eos=-1):
    """(scores, rows, tokens) lists, best first, of each group."""
    groups = x.shape[0] // n_beams
    out = (np.full((groups, k), -np.inf), np.full((groups, k), -1), np.full((groups, k), -1))
    for g in range(groups):
        cands = []
        for row in range(g * n_beams, (g + 1) * n_beams):
            s = np.float64(scores[row])
            if not np.isfinite(s):
                continue
            if finished is not None and finished[row]:
                cands.append((-s, row, 0.0, eos, s))
                continue
            r = x[row].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                m = r.max()
                lse = m + np.log(np.exp(r - m).sum())
            if not np.isfinite(lse):
                continue
            top = np.argsort(-r, kind="stable")[:k]
            cands += [(-(s + (r[t] - lse)), row, -r[t], int(t), s + (r[t] - lse)) for t in top if r[t] > -np.inf]
        for j, c in enumerate(sorted(cands)[:k]):
            out[0][g, j], out[1][g, j], out[2][g, j] = c[4], c[1], c[3]
    return out
