"""Operators for sequences that branch over the paged fp16 key/value cache: attention of a drafted
token tree, forking and compacting of cache pages, and beam search's selection -- their plain forms
in elementary torch operations, the calls of densecore_b200 that compute the same, and the cases
both are timed on.

Cache layout: arena element (page, layer, slot, head, dim) of a tensor
[n_pages * n_layer][16][hkv][128] fp16, page * n_layer + layer first; a block table row lists a
sequence's pages."""
import math

import torch

own = False

PAGE = 16
D = 128
DEV = "cuda"


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one request, a small draft tree on a short chat turn: latency
        dict(name="tree_1x8_ctx200", kind="tree", n_seqs=1, hq=16, hkv=8, n_layer=2, ctx=200, nodes=8, ragged=False),
        # plain chain drafts of a batch (four tokens each), mid contexts, ragged
        dict(name="tree_64x4_ctx2048", kind="tree", n_seqs=64, hq=16, hkv=8, n_layer=1, ctx=2048, nodes=4, ragged=True),
        # the serving batch of the 4B layout with an ordinary tree
        dict(name="tree_32x16_ctx2048", kind="tree", n_seqs=32, hq=32, hkv=8, n_layer=1, ctx=2048, nodes=16, ragged=True),
        # one long document: few rows, a long axis
        dict(name="tree_1x13_ctx100003", kind="tree", n_seqs=1, hq=32, hkv=8, n_layer=1, ctx=100003, nodes=13, ragged=False),
        # large trees at the widest head group: the most arithmetic
        dict(name="tree_16x64_ctx4096", kind="tree", n_seqs=16, hq=64, hkv=8, n_layer=1, ctx=4096, nodes=64, ragged=True),
        # two beam searches of four beams each, 28 layers
        dict(name="fork_2x4_ctx500", kind="fork", groups=2, beams=4, n_layer=28, hkv=8, ctx=500, reserve=1),
        # a serving batch of beam searches, 36 layers
        dict(name="fork_16x4_ctx700", kind="fork", groups=16, beams=4, n_layer=36, hkv=8, ctx=700, reserve=1),
        # an accepted path of one request
        dict(name="compact_1x8", kind="compact", n_seqs=1, n_layer=28, hkv=8, ctx=333, nodes=8),
        # accepted paths of a batch with large trees
        dict(name="compact_32x64", kind="compact", n_seqs=32, n_layer=36, hkv=8, ctx=700, nodes=64),
        # one beam search over a full vocabulary: latency
        dict(name="beam_1x4_v151936", kind="beam", groups=1, beams=4, vocab=151936, k=4, finished=False),
        # an odd vocabulary (rows that do not start on 16 bytes), finished beams, twice as many candidates as beams
        dict(name="beam_7x5_v100003", kind="beam", groups=7, beams=5, vocab=100003, k=10, finished=True),
        # a large batch of wide beams
        dict(name="beam_32x16_v128256", kind="beam", groups=32, beams=16, vocab=128256, k=32, finished=False),
    ]


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "fork", "compact", "beam", "beam"])
    most = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        if kind == "tree":
            hkv = rng.choice([1, 2, 4, 8])
            c = dict(kind="tree", n_seqs=_log(rng, 1, 64), hq=hkv * rng.choice([1, 2, 4, 8]), hkv=hkv,
                     n_layer=rng.choice([1, 2, 3]), ctx=_log(rng, 17, 110000), nodes=_log(rng, 1, 64),
                     ragged=rng.random() < 0.7)
            fits = c["nodes"] <= c["ctx"] and c["n_seqs"] * c["ctx"] * hkv * c["n_layer"] <= 2400000
        elif kind == "fork":
            c = dict(kind="fork", groups=_log(rng, 1, 16), beams=rng.choice([2, 3, 4, 5, 8]),
                     n_layer=rng.choice([16, 28, 36]), hkv=rng.choice([2, 4, 8]), ctx=_log(rng, 5, 700),
                     reserve=rng.choice([0, 1, 1, 9, 40]))
            fits = c["groups"] * c["beams"] <= 64
        elif kind == "compact":
            c = dict(kind="compact", n_seqs=_log(rng, 1, 32), n_layer=rng.choice([16, 28, 36]),
                     hkv=rng.choice([1, 2, 4, 8]), ctx=_log(rng, 65, 900), nodes=_log(rng, 2, 64))
            fits = True
        else:
            beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
            c = dict(kind="beam", groups=_log(rng, 1, 64), beams=beams,
                     vocab=rng.choice([_log(rng, 500, 160000), 128256, 151936]),
                     k=rng.choice([beams, 2 * beams]), finished=rng.random() < 0.4)
            fits = c["groups"] * c["beams"] * c["vocab"] <= 32 * 16 * 128256
        if fits and _cost(c) <= most:
            return c


# ------------------------------------------------------------------- sizes that a case's name fixes
def _spread(lo, hi, n, step):
    """n whole numbers of lo..hi, spread evenly and in mixed order (a batch's ragged lengths)."""
    if n == 1 or lo == hi:
        return [hi] * n
    return [lo + (hi - lo) * ((i * step) % n) // (n - 1) for i in range(n)]


def _tree_sizes(case):
    """(drafted tokens, context with them) of each sequence."""
    n, nodes, ctx = case["n_seqs"], case["nodes"], case["ctx"]
    if not case["ragged"]:
        return [nodes] * n, [ctx] * n
    ns = _spread(max(1, nodes // 2), nodes, n, 7)
    ls = _spread(max(nodes, ctx // 8), ctx, n, 5)
    return ns, ls


def _fork_sizes(case):
    """(context of each row, parent of each row, shared whole pages of each group)."""
    g, b, ctx = case["groups"], case["beams"], case["ctx"]
    lens = [c for c in _spread(max(1, ctx - ctx // 3), ctx, g, 3) for _ in range(b)]
    parents = []
    for i in range(g):
        for j in range(b):   # the better beams have more children, the last ones are dropped
            parents.append(i * b + (j * j) // (2 * b))
    return lens, parents


def _compact_sizes(case):
    """(tokens before the draft, accepted path) of each row: every third node, from the first."""
    n, nodes = case["n_seqs"], case["nodes"]
    base = _spread(max(0, case["ctx"] // 2 - nodes), case["ctx"] - nodes if case["ctx"] > nodes else 0, n, 5)
    paths = [[0] + list(range(1 + i % 3, nodes, 3 + i % 2)) for i in range(n)]
    return base, paths


def work(case):
    """Bytes that have to be read and written once, and the multiply-adds times two."""
    if case["kind"] == "tree":
        ns, ls = _tree_sizes(case)
        b = 2 * 2 * D * case["hkv"] * sum(ls) + 2 * 4 * D * case["hq"] * sum(ns)
        b += 8 * sum(ns) + 4 * sum((c + PAGE - 1) // PAGE for c in ls)
        return {"bytes": b, "flops": 4 * D * case["hq"] * sum(n * c for n, c in zip(ns, ls))}
    if case["kind"] == "fork":
        lens, parents = _fork_sizes(case)
        kids = [parents.count(p) for p in range(len(lens))]
        slots = sum((k - 1) * (n % PAGE) for k, n in zip(kids, lens) if k > 1)
        pages = sum((n + case["reserve"] + PAGE - 1) // PAGE for n in lens)
        return {"bytes": 2 * slots * case["n_layer"] * 2 * case["hkv"] * D * 2 + 2 * 4 * pages + 16 * len(lens), "flops": 0}
    if case["kind"] == "compact":
        _, paths = _compact_sizes(case)
        moved = sum(sum(j != t for j, t in enumerate(p)) for p in paths)
        return {"bytes": 2 * moved * case["n_layer"] * 2 * case["hkv"] * D * 2 + 16 * len(paths), "flops": 0}
    rows = case["groups"] * case["beams"]
    return {"bytes": 4 * rows * case["vocab"] + 4 * rows + 12 * case["groups"] * case["k"], "flops": 2 * rows * case["vocab"]}


# ----------------------------------------------------------------------------------------- inputs
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _random_tree(g, n):
    """Mask bits (as one signed 64-bit word a node) of a random tree: node 0 is the root, node i > 0
    hangs under an earlier node, and each node sees its ancestors and itself."""
    bits = []
    for i in range(n):
        up = 0 if i == 0 else bits[int(torch.randint(0, i, (1,), generator=g))]
        bits.append(up | (1 << i))
    return [b - (1 << 64) if b >> 63 else b for b in bits]


def _arenas(gg, pages, n_layer, hkv):
    shape = (pages * n_layer, PAGE, hkv, D)
    k = torch.empty(shape, dtype=torch.float16, device=DEV).normal_(generator=gg)
    v = torch.empty(shape, dtype=torch.float16, device=DEV).normal_(generator=gg)
    return k, v


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gg = torch.Generator(device=DEV).manual_seed(seed)
    st = dict(case=case)
    if case["kind"] == "tree":
        ns, ls = _tree_sizes(case)
        pages = [(c + PAGE - 1) // PAGE for c in ls]
        order = torch.randperm(sum(pages) + 3, generator=g).to(torch.int32)
        bt = torch.zeros((len(ls), max(pages)), dtype=torch.int32)
        at = 0
        for i, p in enumerate(pages):
            bt[i, :p] = order[at:at + p]
            at += p
        st["k"], st["v"] = _arenas(gg, sum(pages) + 3, case["n_layer"], case["hkv"])
        starts = [0]
        for n in ns:
            starts.append(starts[-1] + n)
        mask = [w for n in ns for w in _random_tree(g, n)]
        st.update(q=torch.randn((starts[-1], case["hq"], D), generator=gg, device=DEV) * 2, bt=bt.to(DEV),
                  starts=_ints(starts), ctx=_ints(ls), layer=case["n_layer"] - 1, max_nodes=max(ns), max_ctx=max(ls),
                  mask=torch.tensor(mask, dtype=torch.int64, device=DEV).view(-1, 1))
    elif case["kind"] == "fork":
        lens, parents = _fork_sizes(case)
        rows, b = len(lens), case["beams"]
        total = [(n + PAGE - 1) // PAGE for n in lens]
        width = max((n + case["reserve"] + PAGE - 1) // PAGE for n in lens) + 1
        taken = sum(t - (t // 2 if r % b else 0) for r, t in enumerate(total))
        most = 1 + taken + rows * (2 + case["reserve"] // PAGE) + 8
        order = torch.randperm(most - 1, generator=g).add(1).to(torch.int32).tolist()  # page 0 is the idle page
        bt = torch.zeros((rows, width), dtype=torch.int32)
        refs = torch.zeros(most, dtype=torch.int32)
        refs[0] = 1
        at = 0
        for r in range(rows):   # a group's beams share their first pages (the prompt), the rest is their own
            shared = total[r] // 2
            for j in range(total[r]):
                if j < shared and r % b:
                    bt[r, j] = bt[r - r % b, j]
                else:
                    bt[r, j] = order[at]
                    at += 1
                refs[bt[r, j]] += 1
        st["k"], st["v"] = _arenas(gg, most, case["n_layer"], case["hkv"])
        shuffled = [i * b + j for i in range(case["groups"]) for j in torch.randperm(b, generator=g).tolist()]
        st.update(bt=bt.to(DEV), refs=refs.to(DEV), lens=_ints(lens), pages=_ints(total),
                  parents=_ints([shuffled[p] for p in parents]), reserve=_ints([case["reserve"]] * rows))
    elif case["kind"] == "compact":
        base, paths = _compact_sizes(case)
        pages = [(c + case["nodes"] + PAGE - 1) // PAGE for c in base]
        order = torch.randperm(sum(pages), generator=g).to(torch.int32)
        bt = torch.zeros((len(base), max(pages)), dtype=torch.int32)
        at = 0
        for i, p in enumerate(pages):
            bt[i, :p] = order[at:at + p]
            at += p
        st["k"], st["v"] = _arenas(gg, sum(pages), case["n_layer"], case["hkv"])
        path = torch.zeros((len(base), max(len(p) for p in paths)), dtype=torch.int32)
        for i, p in enumerate(paths):
            path[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
        st.update(bt=bt.to(DEV), base=_ints(base), path=path.to(DEV), path_lens=_ints([len(p) for p in paths]),
                  ctx=torch.zeros(len(base), dtype=torch.int32, device=DEV))
    else:
        rows = case["groups"] * case["beams"]
        x = torch.randn((rows, case["vocab"]), generator=gg, device=DEV) * 2.5
        few = torch.randint(0, case["vocab"], (rows, 6), generator=gg, device=DEV)   # the few likely tokens of a model's step
        x.scatter_add_(1, few, torch.rand((rows, 6), generator=gg, device=DEV) * 12)
        st.update(x=x, scores=-torch.rand(rows, generator=gg, device=DEV) * 6, finished=None, eos=case["vocab"] // 2)
        if case["finished"]:
            st["finished"] = (torch.rand(rows, generator=gg, device=DEV) < 0.3).to(torch.uint8)
    return st


# ------------------------------------------------------------------------------------ plain forms
def _plain_tree(st):
    case, dev = st["case"], st["q"].device
    hkv, nl = case["hkv"], case["n_layer"]
    nrep = case["hq"] // hkv
    n_seqs, width = st["bt"].shape
    at = st["bt"].long() * nl + st["layer"]
    ctx, starts = st["ctx"].long(), st["starts"].long()
    ns = starts[1:] - starts[:-1]
    key = torch.arange(width * PAGE, device=dev)
    there = key < ctx[:, None]
    k = st["k"][at].reshape(n_seqs, -1, hkv, D).float().permute(0, 2, 3, 1)
    v = st["v"][at].reshape(n_seqs, -1, hkv, D).float()
    v = torch.where(there[:, :, None, None], v, 0.0).permute(0, 2, 1, 3)
    node = torch.arange(st["max_nodes"], device=dev)
    row = (starts[:-1, None] + node).clamp(max=st["q"].shape[0] - 1)      # [seq, node]
    q = st["q"][row].view(n_seqs, -1, hkv, nrep, D).permute(0, 2, 1, 3, 4).reshape(n_seqs, hkv, -1, D)
    s = torch.matmul(q, k) * (1.0 / D ** 0.5)
    j = key - (ctx - ns)[:, None]                                        # drafted token of a key; < 0: history
    words = st["mask"][row]                                              # [seq, node, words]
    word = torch.gather(words, 2, (j.clamp(0, 64 * words.shape[2] - 1) // 64)[:, None, :].expand(-1, words.shape[1], -1))
    bit = (word >> (j % 64)[:, None, :]) & 1
    seen = ((j < 0)[:, None, :] | (bit == 1)) & there[:, None, :]        # [seq, node, key]
    seen = seen[:, None, :, None, :].expand(-1, hkv, -1, nrep, -1).reshape(s.shape)
    s = torch.where(seen, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    del s, seen
    norm = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(norm > 0, norm, 1.0)
    o = o.view(n_seqs, hkv, -1, nrep, D).permute(0, 2, 1, 3, 4).reshape(n_seqs, -1, case["hq"], D)
    token = torch.arange(st["q"].shape[0], device=dev)
    seq = (token[:, None] >= starts[None, 1:]).sum(1)
    return o[seq, token - starts[seq]]


def _plain_fork(st):
    bt, refs, lens, pages = st["bt"], st["refs"], st["lens"], st["pages"]
    dev = bt.device
    col = torch.arange(bt.shape[1], device=dev)
    n = lens.shape[0]
    new = refs.clone().index_add_(0, bt.flatten(), -(col < pages[:, None]).flatten().int())
    live = st["parents"] >= 0
    p = st["parents"].clamp(min=0).long()
    ln = torch.where(live, lens[p], 0)
    used = (ln + PAGE - 1) // PAGE
    t = bt[p]
    new.index_add_(0, t.flatten(), (col < used[:, None]).flatten().int())
    part = ln % PAGE != 0
    last = (used - 1).clamp(min=0).long()
    src = t.gather(1, last[:, None])[:, 0]
    earlier = (src[None, :] == src[:, None]) & part[None, :] & (torch.arange(n, device=dev)[None, :] < torch.arange(n, device=dev)[:, None])
    copied = part & (new[src.long()] - earlier.sum(1) > 1)
    total = torch.where(live, (ln + st["reserve"] + PAGE - 1) // PAGE, 0)
    asks = copied.int() + (total - used)
    first = torch.cumsum(asks, 0) - asks
    free = torch.argsort((new != 0).int(), stable=True).to(torch.int32)   # free pages first, ascending
    short = (asks.sum() - (new == 0).sum()).clamp(min=0).int()
    new.index_add_(0, src, -copied.int())
    rank = first[:, None] + copied[:, None] + (col - used[:, None])
    fresh = (col >= used[:, None]) & (col < total[:, None])
    t = torch.where(fresh, free[rank.clamp(0, free.shape[0] - 1).long()], t)
    dst = free[first.clamp(0, free.shape[0] - 1).long()]
    t = torch.where(copied[:, None] & (col == last[:, None]), dst[:, None], t)
    new[free] = torch.where(torch.arange(free.shape[0], device=dev) < asks.sum(), 1, new[free])
    t = torch.where(col < total[:, None], t, torch.where(col < pages[:, None], 0, bt))
    if int(short) == 0:
        at = copied.nonzero()[:, 0]
        slot = torch.arange(PAGE, device=dev)[None, None, :, None, None] < (ln % PAGE)[at][:, None, None, None, None]
        for a in (st["k"], st["v"]):
            a = a.view(refs.shape[0], -1, *a.shape[1:])
            a[dst[at].long()] = torch.where(slot, a[src[at].long()], a[dst[at].long()])
        bt.copy_(t)
        refs.copy_(new)
        lens.copy_(ln)
        pages.copy_(total)
    return dict(k=st["k"], v=st["v"], tables=bt, refs=refs, lens=lens, pages=pages, short=short)


def _plain_compact(st):
    bt, nl = st["bt"], st["case"]["n_layer"]
    j = torch.arange(st["path"].shape[1], device=bt.device)
    row, at = ((j < st["path_lens"][:, None]) & (st["path"] != j)).nonzero(as_tuple=True)
    src = (st["base"][row] + st["path"][row, at]).long()
    dst = (st["base"][row] + at).long()
    for a in (st["k"], st["v"]):
        a = a.view(-1, nl, *a.shape[1:])
        a[bt[row, dst // PAGE].long(), :, dst % PAGE] = a[bt[row, src // PAGE].long(), :, src % PAGE]
    st["ctx"].copy_(st["base"] + st["path_lens"])
    return dict(k=st["k"], v=st["v"], ctx=st["ctx"])


def _plain_beam(st):
    case, x = st["case"], st["x"].double()    # scores of two beams may lie next to each other
    m = x.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(1, keepdim=True))
    s = st["scores"].double()[:, None]
    c = torch.where(torch.isfinite(lse) & torch.isfinite(s), s + (x - lse), -math.inf)
    if st["finished"] is not None:
        alone = torch.arange(x.shape[1], device=x.device)[None, :] == st["eos"]
        alone = torch.where(alone & torch.isfinite(s), s, -math.inf)
        c = torch.where(st["finished"][:, None] != 0, alone, c)
    value, at = torch.sort(c.view(case["groups"], -1), dim=1, descending=True, stable=True)
    value, at = value[:, :case["k"]], at[:, :case["k"]]
    first = torch.arange(case["groups"], device=x.device)[:, None] * case["beams"]
    none = value == -math.inf
    row = torch.where(none, -1, first + at // case["vocab"])
    token = torch.where(none, -1, at % case["vocab"])
    return dict(scores=value.float(), rows=row.int(), tokens=token.int())


# -------------------------------------------------------------------------- the framework's calls
def _own_tree(st):
    from densecore_b200 import ops
    case = st["case"]
    if "ws" not in st:   # a program keeps its workspace and output over its steps
        st["ws"] = torch.empty(ops.paged_attn_tree_scratch_size(st["ctx"].numel(), case["hq"], case["hkv"], st["max_nodes"], st["max_ctx"]),
                               dtype=torch.uint8, device=st["q"].device)
        st["out"] = torch.empty_like(st["q"])
    return ops.paged_attn_tree(st["q"], st["k"], st["v"], case["n_layer"], st["layer"], st["bt"], st["starts"], st["ctx"], st["mask"],
                               case["hkv"], st["max_nodes"], st["max_ctx"], out=st["out"], scratch=st["ws"])


def _own_fork(st):
    from densecore_b200 import ops
    if "ws" not in st:
        st["ws"] = torch.empty(ops.kv_fork_scratch_size(st["bt"].shape[0], st["bt"].shape[1], st["refs"].numel()), dtype=torch.uint8, device=st["bt"].device)
        st["status"] = torch.empty((), dtype=torch.int32, device=st["bt"].device)
    short = ops.kv_fork(st["k"], st["v"], st["case"]["n_layer"], st["bt"], st["lens"], st["pages"], st["refs"], st["parents"],
                        reserve=st["reserve"], fill_page=0, status=st["status"], scratch=st["ws"])
    return dict(k=st["k"], v=st["v"], tables=st["bt"], refs=st["refs"], lens=st["lens"], pages=st["pages"], short=short)


def _own_compact(st):
    from densecore_b200 import ops
    ops.kv_compact(st["k"], st["v"], st["case"]["n_layer"], st["bt"], st["base"], st["path"], st["path_lens"], st["ctx"])
    return dict(k=st["k"], v=st["v"], ctx=st["ctx"])


def _own_beam(st):
    from densecore_b200 import ops
    case = st["case"]
    if "ws" not in st:
        dev = st["x"].device
        st["ws"] = torch.empty(ops.beam_select_scratch_size(case["groups"], case["beams"], case["vocab"], case["k"]), dtype=torch.uint8, device=dev)
        shape = (case["groups"], case["k"])
        st["out"] = (torch.empty(shape, device=dev), torch.empty(shape, dtype=torch.int32, device=dev), torch.empty(shape, dtype=torch.int32, device=dev))
    s, r, t = ops.beam_select(st["x"], st["scores"], case["beams"], case["k"], finished=st["finished"], eos=st["eos"], out=st["out"], scratch=st["ws"])
    return dict(scores=s, rows=r, tokens=t)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"tree": _own_tree, "fork": _own_fork, "compact": _own_compact, "beam": _own_beam}[kind](state)
    return {"tree": _plain_tree, "fork": _plain_fork, "compact": _plain_compact, "beam": _plain_beam}[kind](state)


# ------------------------------------------------------------ the definitions, in 64 bits, by loops
def _exact_tree(st):
    case = st["case"]
    nrep, nl = case["hq"] // case["hkv"], case["n_layer"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    starts, ctx, masks = st["starts"].tolist(), st["ctx"].tolist(), st["mask"].tolist()
    for s, n_keys in enumerate(ctx):
        a, b = starts[s], starts[s + 1]
        rows = st["bt"][s, :(n_keys + PAGE - 1) // PAGE].long() * nl + st["layer"]
        k = st["k"][rows].reshape(-1, case["hkv"], D)[:n_keys].double()
        v = st["v"][rows].reshape(-1, case["hkv"], D)[:n_keys].double()
        hist = n_keys - (b - a)
        seen = torch.ones((b - a, n_keys), dtype=torch.bool)
        for i in range(b - a):
            for t in range(b - a):
                seen[i, hist + t] = bool((masks[a + i][t // 64] >> (t % 64)) & 1)
        bias = torch.zeros(seen.shape, dtype=torch.float64).masked_fill_(~seen, -math.inf).to(DEV)
        for h in range(case["hq"]):
            e = torch.einsum("id,jd->ij", st["q"][a:b, h].double(), k[:, h // nrep]) / math.sqrt(D) + bias
            out[a:b, h] = torch.softmax(e, -1).nan_to_num(0.0) @ v[:, h // nrep]
    return out


def _exact_fork(st):
    t, refs, lens, held = st["bt"].tolist(), st["refs"].tolist(), st["lens"].tolist(), st["pages"].tolist()
    parents, reserve = st["parents"].tolist(), st["reserve"].tolist()
    for i, n in enumerate(held):
        for j in range(n):
            refs[t[i][j]] -= 1
    rows, ln, dst = [], [], []
    for p in parents:
        ln.append(lens[p] if p >= 0 else 0)
        rows.append(t[p][:(ln[-1] + PAGE - 1) // PAGE] if p >= 0 else [])
        for b in rows[-1]:
            refs[b] += 1
    free = iter([b for b, r in enumerate(refs) if r == 0])
    k, v = (st[a].view(len(refs), st["case"]["n_layer"], PAGE, -1) for a in ("k", "v"))
    for i, p in enumerate(parents):
        if ln[i] % PAGE and refs[rows[i][-1]] > 1:
            b = next(free)
            for a in (k, v):
                a[b, :, :ln[i] % PAGE] = a[rows[i][-1], :, :ln[i] % PAGE]
            refs[rows[i][-1]] -= 1
            refs[b] = 1
            rows[i][-1] = b
        while p >= 0 and len(rows[i]) * PAGE < ln[i] + reserve[i]:
            rows[i].append(next(free))
            refs[rows[i][-1]] = 1
    for i, r in enumerate(rows):
        tail = [0 if j < held[i] else t[i][j] for j in range(len(r), len(t[i]))]
        t[i] = r + tail
    return dict(k=st["k"].double(), v=st["v"].double(), tables=_ints(t), refs=_ints(refs), lens=_ints(ln), pages=_ints([len(r) for r in rows]), short=0)


def _exact_compact(st):
    t, base, path = st["bt"].tolist(), st["base"].tolist(), st["path"].tolist()
    k, v = (st[a].view(-1, st["case"]["n_layer"], PAGE, st["case"]["hkv"] * D) for a in ("k", "v"))
    ctx = []
    for i, n in enumerate(st["path_lens"].tolist()):
        for j in range(n):
            src, dst = base[i] + path[i][j], base[i] + j
            for a in (k, v):
                a[t[i][dst // PAGE], :, dst % PAGE] = a[t[i][src // PAGE], :, src % PAGE].clone()
        ctx.append(base[i] + n)
    return dict(k=st["k"].double(), v=st["v"].double(), ctx=_ints(ctx))


def _exact_beam(st):
    case = st["case"]
    out = torch.full((case["groups"], case["k"]), -math.inf, dtype=torch.float64, device=DEV)
    for g in range(case["groups"]):
        cands = []
        for b in range(g * case["beams"], (g + 1) * case["beams"]):
            s = st["scores"][b].double()
            if st["finished"] is not None and int(st["finished"][b]):
                cands.append(s.view(1))
            else:
                x = st["x"][b].double()
                cands.append(s + torch.topk(x, min(case["k"], x.numel())).values - torch.logsumexp(x, 0))
        best = torch.cat(cands).sort(descending=True).values[:case["k"]]
        out[g, :best.numel()] = best
    return dict(scores=out, rows=None, tokens=None)


def exact(case, seed):
    st = prepare(case, seed)
    return {"tree": _exact_tree, "fork": _exact_fork, "compact": _exact_compact, "beam": _exact_beam}[case["kind"]](st)
