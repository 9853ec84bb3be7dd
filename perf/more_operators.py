"""Four operators of a speculative decode step over a paged cache, as cases that can be timed and compared.

``tree``    ``ops.draft_tree``: what the nodes of drafted trees see, the positions that they are rotated by and the places that they take in the cache
``attend``  ``ops.paged_tree_attention``: the nodes of a tree per sequence against the pages of its context and the nodes before them
``verify``  ``ops.verify_drafts``: which drafted tokens the target's probabilities accept, from given random numbers, and the token that follows
``move``    ``ops.paged_move``: rows of a paged cache to other places, in all layers: the accepted path closed up, the tail of a forked sequence

With ``own`` false ``run`` computes them in elementary torch operations, in 32 bits rounded once (in 64 where a comparison decides); with ``own``
true through the package's entry points.  ``exact`` computes the same from the definitions in 64 bits.  Head counts, head widths, windows and
vocabularies are those of the repository's configurations, tests and benchmark, or generic.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
SCALE = 0.12                 # the framework's softmax scale
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # One sequence with a small tree: a launch.
        dict(name="tree_b1", kind="tree", B=1, T=8, shape="random", ragged=False, max_len=8192, empty=0),
        # A large batch of the largest trees of unequal size, free slots among them.
        dict(name="tree_b512_256", kind="tree", B=512, T=256, shape="random", ragged=True, max_len=8192, empty=17),
        # The generator's layer and default cache type, one sequence, a chain of drafted tokens: latency and the split over the context.
        dict(name="attend_b1_chain", kind="attend", B=1, T=8, shape="chain", ragged=False, Hq=12, H=12, D=128, page=64, min_len=8000, max_len=8000, window=0,
             cache="float16", empty=0),
        # A batch of chats of unequal length under a sliding window, trees of unequal size, free slots among them.
        dict(name="attend_b24_window_4096", kind="attend", B=24, T=16, shape="random", ragged=True, Hq=16, H=16, D=128, page=16, min_len=1, max_len=8300, window=4096,
             cache="bfloat16", empty=3),
        # Eight query heads to a key head and trees of 32: 256 queries for every key that is read.
        dict(name="attend_shared_heads_b12", kind="attend", B=12, T=32, shape="random", ragged=False, Hq=64, H=8, D=128, page=64, min_len=100, max_len=24000, window=0,
             cache="bfloat16", empty=0),
        # Two contexts near the end of the rotary tables, four tokens drafted: reading the cache is all there is.
        dict(name="attend_b2_131000", kind="attend", B=2, T=5, shape="chain", ragged=False, Hq=16, H=16, D=128, page=128, min_len=130900, max_len=131000, window=0,
             cache="bfloat16", empty=0),
        # One sequence's tree of chosen tokens, the vocabulary of the generator's model.
        dict(name="verify_b1", kind="verify", B=1, T=8, shape="random", ragged=False, V=50304, logits="float32", temperature="one", kept=0, draft=False, int32=False),
        # A batch of requests with temperatures of their own behind a filter that has left few tokens, trees of unequal size, an odd vocabulary.
        dict(name="verify_b32_filtered", kind="verify", B=32, T=16, shape="random", ragged=True, V=50257, logits="float32", temperature="rows", kept=64, draft=False,
             int32=False),
        # A large batch of chains drawn from a draft model's distributions, a large vocabulary, bf16 logits.
        dict(name="verify_b64_drawn", kind="verify", B=64, T=5, shape="chain", ragged=False, V=131072, logits="bfloat16", temperature="one", kept=0, draft=True, int32=True),
        # One sequence of the generator's stack: the accepted nodes of its tree become the context's next positions.
        dict(name="move_accepted_b1", kind="move", B=1, T=16, L=12, H=12, D=128, page=64, max_len=4000, cache="float16", fork=False, rows=5),
        # The same for a batch, in a deeper stack with shared heads.
        dict(name="move_accepted_b64", kind="move", B=64, T=32, L=32, H=8, D=128, page=16, max_len=3000, cache="bfloat16", fork=False, rows=9),
        # Branches of a few sequences: the pages before the last are shared, the rows of the last one copied.
        dict(name="move_forked_b96", kind="move", B=96, T=0, L=12, H=16, D=128, page=64, max_len=2000, cache="bfloat16", fork=True, rows=63),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    kind = rng.choice(["tree", "attend", "attend", "attend", "verify", "verify", "verify", "move", "move"])
    shape = rng.choice(["chain", "random", "random", "wide"])
    if kind == "tree":
        B = _log_int(rng, 1, 512)
        return dict(kind=kind, B=B, T=_log_int(rng, 1, 256), shape=shape, ragged=rng.random() < 0.5, max_len=_log_int(rng, 1, 131072), empty=rng.choice([0, 0, B // 8]))
    if kind == "verify":
        draft = rng.random() < 0.4
        return dict(kind=kind, B=_log_int(rng, 1, 128), T=_log_int(rng, 1, 64), shape=shape, ragged=rng.random() < 0.5, V=_log_int(rng, 300, 200000),
                    logits=rng.choice(["float32", "bfloat16", "float16"]), temperature=rng.choice(["one", "rows"] if draft else ["none", "one", "one", "rows"]),
                    kept=rng.choice([0, 0, 64]), draft=draft, int32=rng.random() < 0.5)
    D = rng.choice([64, 128, 128, 256])
    H = rng.choice([1, 2, 4, 8, 12, 16])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    cache = rng.choice(["bfloat16", "bfloat16", "float16"])
    if kind == "attend":
        B, T = _log_int(rng, 1, 256), _log_int(rng, 1, 64)
        max_len = _log_int(rng, 1, 131000)
        return dict(kind=kind, B=B, T=T, shape=shape, ragged=rng.random() < 0.5, Hq=H * rng.choice([1, 1, 1, 2, 4, 8]), H=H, D=D, page=page,
                    min_len=max(0, rng.choice([max_len, max_len // 2, max_len // 100])), max_len=max_len, window=rng.choice([0, 0, _log_int(rng, 1, max_len)]),
                    cache=cache, empty=rng.choice([0, 0, B // 8]))
    fork = rng.random() < 0.4
    T = 0 if fork else _log_int(rng, 2, 256)
    return dict(kind=kind, B=_log_int(rng, 1, 96), T=T, L=_log_int(rng, 1, 48), H=H, D=D, page=page, max_len=_log_int(rng, 300, 4000), cache=cache, fork=fork,
                rows=_log_int(rng, 1, page - 1) if fork else _log_int(rng, 1, min(T, 32)))


def draw(rng):
    """One more case of the ranges above; none costs more than the largest listed one."""
    while True:
        case = _draw_once(rng)
        w = work(case)
        if w["bytes"] > 2.1e9 or w["flops"] > 7e10:
            continue
        if case["kind"] == "attend" and (case["B"] * case["T"] * case["max_len"] * case["Hq"] > 6e8 or case["B"] * case["max_len"] * case["H"] * case["D"] > 6e8):
            continue                                                          # the plain form's scores, its copy of the keys
        if case["kind"] == "verify" and case["B"] * case["T"] * case["V"] > 5e7:
            continue
        if case["kind"] == "move" and _pool_bytes(case) > 8e9:
            continue
        return case


def _case_rng(case):
    return random.Random(case["B"] * 1000003 + case["T"] * 131 + case.get("max_len", 0))


def _context(case):
    """Positions ahead of each sequence's tree (the same for every seed): spread over the range on a logarithmic scale, the longest among them; -1 for
    ``empty`` slots without a sequence."""
    rng, lo = _case_rng(case), case.get("min_len", 1)
    lens = [_log_int(rng, max(1, lo), max(1, case["max_len"])) - (1 if lo == 0 else 0) for _ in range(case["B"])]
    lens[rng.randrange(case["B"])] = case["max_len"]
    for b in rng.sample(range(case["B"]), min(case.get("empty", 0), case["B"] - 1)):
        lens[b] = -1
    return lens


def _nodes(case):
    rng = _case_rng(case)
    rng.random()
    return [rng.randint(1, case["T"]) if case["ragged"] else case["T"] for _ in range(case["B"])]


def _visible(case):
    """Keys of each sequence that some node of it sees, and pairs of a node and a key that it sees at most."""
    keys, pairs = 0, 0
    for n, t in zip(_context(case), _nodes(case)):
        if n >= 0:
            k = min(n, case["window"]) + t if case["window"] else n + t
            keys, pairs = keys + k, pairs + k * t
    return keys, pairs


def _moved(case):
    """Source rows of every sequence, relative to where the first one goes: an accepted path, or the rows of a page's beginning."""
    rng = _case_rng(case)
    if case["fork"]:
        return [list(range(rng.randint(1, case["rows"]))) for _ in range(case["B"])]
    return [[0] + sorted(rng.sample(range(1, case["T"]), rng.randint((case["rows"] + 1) // 2, case["rows"]) - 1)) for _ in range(case["B"])]


def _pool_bytes(case):
    pages = case["B"] * (-(-(case["rows"] + case["T"]) // case["page"]) + 1)
    return 4 * pages * case["L"] * case["H"] * case["page"] * case["D"]


def work(case):
    B, T = case["B"], case["T"]
    if case["kind"] == "tree":
        return {"bytes": 4 * B * T + 8 * B + 4 * B * T * (-(-T // 32) + 3), "flops": B * T}
    if case["kind"] == "attend":
        keys, pairs = _visible(case)
        return {"bytes": 4 * keys * case["H"] * case["D"] + 4 * sum(_nodes(case)) * case["Hq"] * case["D"] + 4 * B * T * -(-T // 32) + 4 * keys // case["page"],
                "flops": 4 * pairs * case["Hq"] * case["D"]}
    if case["kind"] == "verify":
        rows, size = sum(_nodes(case)), 4 if case["logits"] == "float32" else 2
        greedy = case["temperature"] == "none"
        return {"bytes": rows * case["V"] * (size + (4 if case["draft"] else 0)) + (0 if greedy else 4 * B * case["V"]) + 16 * B * T, "flops": 4 * rows * case["V"]}
    rows = sum(1 for path in _moved(case) for i, j in enumerate(path) if case["fork"] or i != j)
    return {"bytes": max(16, 8 * rows * case["L"] * case["H"] * case["D"]), "flops": 1}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _parents(case, rng):
    """Trees as lists of parents; node 0 is the root.  ``wide``: most nodes are children of the first few."""
    T = case["T"]
    if case["shape"] == "chain":
        return [[i - 1 for i in range(T)] for _ in range(case["B"])]
    if case["shape"] == "wide":
        return [[-1] + [rng.randrange(min(i, 3)) for i in range(1, T)] for _ in range(case["B"])]
    return [[-1] + [rng.randrange(max(0, i - 5), i) for i in range(1, T)] for _ in range(case["B"])]


def _table(entries, width, g):
    """int32 [S, width] with pages of a shuffled pool at the entries named (lists of entries, one per sequence), -1 elsewhere; and the pool's size."""
    total = sum(len(e) for e in entries)
    pages = torch.randperm(total + 3, generator=g, device=DEVICE)[:total].to(torch.int32).cpu()
    table = torch.full((len(entries), width), -1, dtype=torch.int32)
    at = 0
    for s, e in enumerate(entries):
        table[s, e] = pages[at:at + len(e)]
        at += len(e)
    return table.to(DEVICE), total + 3


def prepare(case, seed):
    g, rng = torch.Generator(device=DEVICE).manual_seed(seed), random.Random(seed)
    return {"tree": _prepare_tree, "attend": _prepare_attend, "verify": _prepare_verify, "move": _prepare_move}[case["kind"]](case, g, rng)


def _prepare_tree(case, g, rng):
    lens = [n if n < 0 else max(0, n - rng.randrange(64)) for n in _context(case)]
    return dict(kind="tree", parents=_ints(_parents(case, rng)), lens=_ints(lens), nodes=_ints(_nodes(case)) if case["ragged"] else None)


def _prepare_attend(case, g, rng):
    lens, nodes, parents = _context(case), _nodes(case), _parents(case, rng)
    B, T, H, D, page = case["B"], case["T"], case["H"], case["D"], case["page"]
    entries = [[] if n < 0 else list(range((max(0, n + 1 - case["window"]) if case["window"] else 0) // page, -(-(n + t) // page))) for n, t in zip(lens, nodes)]
    table, pool = _table(entries, -(-(case["max_len"] + T) // page), g)
    masks = []
    for of in parents:
        seen = []
        for i, p in enumerate(of):
            seen.append((1 << i) | (seen[p] if p >= 0 else 0))
        masks.append([[(m >> 32 * w & 0xffffffff) - ((m >> 32 * w + 31 & 1) << 32) for w in range(-(-T // 32))] for m in seen])
    cache = DTYPES[case["cache"]]
    return dict(kind="attend", q=_randn(g, B, T, case["Hq"], D, dtype=cache), table=table, k_pages=_randn(g, pool, H, page, D, dtype=cache),
                v_pages=_randn(g, pool, H, page, D, dtype=cache), lens=_ints(lens), nodes=_ints(nodes) if case["ragged"] else None, mask=_ints(masks),
                window=case["window"] or None)


def _prepare_verify(case, g, rng):
    B, T, V = case["B"], case["T"], case["V"]
    parents, nodes = _ints(_parents(case, rng)), _ints(_nodes(case)) if case["ragged"] else None
    logits = _randn(g, B, T, V, dtype=torch.float32).mul_(4)
    tokens = torch.randint(V, (B, T), generator=g, device=DEVICE)
    of, b = parents.clamp(min=0).long(), torch.arange(B, device=DEVICE)[:, None]
    draft = None
    if case["draft"]:                     # the draft model's distributions are near the target's, each node drawn from that of its parent
        draft = torch.softmax(logits + _randn(g, B, T, V, dtype=torch.float32), -1)
        for i in range(1, T):
            row = draft[b[:, 0], of[:, i]]
            tokens[:, i] = (row / torch.empty_like(row).exponential_(generator=g)).argmax(-1)
    else:                                 # the nodes are tokens that a draft has chosen, and that the target finds likely
        # (by parent and token, so that the same child twice is no race)
        logits[b, of, tokens] = 4 * math.sqrt(2 * math.log(V)) + _randn(g, B, T, dtype=torch.float32).gather(1, of) + torch.sin(tokens.float())
    if case["kept"]:
        least = logits.topk(min(case["kept"], V), dim=-1).values[..., -1:]
        logits = logits.masked_fill(logits < least, -math.inf)
    t = {"none": 0.0, "one": 0.8, "rows": None}[case["temperature"]]
    if t is None:
        t = 0.5 + 0.7 * torch.rand(B, generator=g, device=DEVICE)
        if not case["draft"] and B > 3:
            t[B // 3] = 0.0               # one request of the batch takes the likeliest token
    uniform = torch.rand(B, V, generator=g, device=DEVICE).clamp_(min=1e-6)
    some = isinstance(t, torch.Tensor) or t > 0
    return dict(kind="verify", logits=logits.to(DTYPES[case["logits"]]), tokens=tokens.int() if case["int32"] else tokens, parents=parents, nodes=nodes, temperature=t,
                accept=torch.rand(B, T, generator=g, device=DEVICE) if some else None, noise=uniform.log_().neg_().log_().neg_() if some else None, draft=draft)


def _prepare_move(case, g, rng):
    B, page, moved = case["B"], case["page"], _moved(case)
    counts = [len(m) for m in moved]
    cache = DTYPES[case["cache"]]
    room, rng = range(0, case["max_len"] - case["rows"] - case["T"]), _case_rng(case)      # (where sequences are is the case's, what lies there the seed's)
    index = sources = source_starts = None
    if case["fork"]:                      # the new sequences are rows of the table behind those that they come from
        start = [p - p % page for p in (rng.choice(room) for _ in range(B))]
        entries, first = [[] for _ in range(2 * B)], [rng.randrange(B // 3 + 1) for _ in range(B)]
        for b in range(B):
            entries[first[b]] = sorted({*entries[first[b]], start[b] // page})
            entries[B + b] = [start[b] // page]
        starts, counts, sources = [0] * B + start, [0] * B + counts, _ints(list(range(B)) + first)
    else:
        starts = [rng.choice(room) for _ in range(B)]
        entries = [list(range(p // page, (p + case["T"] - 1) // page + 1)) for p in starts]
        index = torch.full((B, case["T"]), -1, dtype=torch.int32)
        for row, m in zip(index, moved):
            row[:len(m)] = torch.tensor(m)
        index = index.to(DEVICE)
    table, pool = _table(entries, -(-case["max_len"] // page), g)
    shape = (case["L"], pool, case["H"], page, case["D"])
    return dict(kind="move", k_pages=_randn(g, *shape, dtype=cache), v_pages=_randn(g, *shape, dtype=cache), table=table, starts=_ints(starts), counts=_ints(counts),
                index=index, sources=sources, rows=max(counts))


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return {"tree": _own_tree, "attend": _own_attend, "verify": _own_verify, "move": _own_move}[state["kind"]](state)
    return {"tree": _plain_tree, "attend": _plain_attend, "verify": _plain_verify, "move": _plain_move}[state["kind"]](state)


def _own_tree(s):
    from daisy_amd import ops
    tree = ops.draft_tree(s["parents"], s["lens"], nodes=s["nodes"])
    return {"mask": tree.mask, "positions": tree.positions, "slots": tree.slots}


def _own_attend(s):
    from daisy_amd import ops
    return ops.paged_tree_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["mask"], nodes=s["nodes"], window=s["window"], scale=SCALE)


def _own_verify(s):
    from daisy_amd import ops
    path, counts, token = ops.verify_drafts(s["logits"], s["tokens"], s["parents"], nodes=s["nodes"], temperature=s["temperature"], accept=s["accept"],
                                            noise=s["noise"], draft=s["draft"])
    return {"path": path, "counts": counts, "token": token}


def _own_move(s):
    from daisy_amd import ops
    ops.paged_move(s["k_pages"], s["v_pages"], s["table"], s["starts"], s["counts"], rows=s["rows"], index=s["index"], sources=s["sources"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _there(s, B, T):
    """Which nodes there are, bool [B, T]."""
    i = torch.arange(T, device=DEVICE)
    there = torch.ones(B, T, dtype=torch.bool, device=DEVICE) if s["nodes"] is None else i[None] < s["nodes"][:, None]
    return there & (s["lens"][:, None] >= 0) if "lens" in s else there


def _ancestors(parents):
    """bool [B, T, T]: node i is node j or comes from it."""
    B, T = parents.shape
    i = torch.arange(T, device=DEVICE)
    seen = torch.eye(T, dtype=torch.bool, device=DEVICE).expand(B, T, T)
    up = torch.where((parents >= 0) & (parents < i[None]), parents.long(), i[None])      # (a root is its own parent here)
    for _ in range(max(1, (T - 1).bit_length())):
        seen = seen | seen.gather(1, up[:, :, None].expand(B, T, T))
        up = up.gather(1, up)
    return seen


def _plain_tree(s):
    B, T = s["parents"].shape
    there, i = _there(s, B, T), torch.arange(T, device=DEVICE)
    seen = _ancestors(s["parents"])
    depth = seen.sum(-1) - 1
    words = torch.zeros(B, T, -(-T // 32) * 32, dtype=torch.bool, device=DEVICE)
    words[..., :T] = seen & there[:, :, None]
    total = (words.view(B, T, -1, 32).long() << torch.arange(32, device=DEVICE)).sum(-1)
    position, slot = (torch.where(there, s["lens"][:, None] + x, -1).int().flatten() for x in (depth, i[None]))
    return {"mask": (total - ((total >> 31) << 32)).int(), "positions": position, "slots": slot}


def _plain_attend(s):
    q, table, lens = s["q"], s["table"], s["lens"][:, None]
    B, T, Hq, D = q.shape
    H, page = s["k_pages"].shape[1:3]
    L = table.size(1) * page
    i, t = torch.arange(T, device=DEVICE), torch.arange(L, device=DEVICE)
    there = _there(s, B, T)
    bits = (s["mask"][:, :, i >> 5] >> (i & 31) & 1).bool() & there[:, None, :]
    # every key's node, the bit of which decides; what stays of the last `window`: those with fewer than that many behind them
    node = t[None] - lens
    of_tree = (node >= 0) & (node < T)
    seen = torch.where((node < 0)[:, None], True, bits.gather(2, node.clamp(0, T - 1)[:, None].expand(B, T, L)) & of_tree[:, None]) & there[:, :, None]
    if s["window"]:
        behind = seen.flip(-1).cumsum(-1, dtype=torch.int32).flip(-1)
        seen = seen & (behind <= s["window"])
    pages = table.clamp(min=0).long()
    k = s["k_pages"][pages].float().transpose(1, 2).reshape(B, H, L, D)
    scores = torch.matmul(q.float().reshape(B, T, H, Hq // H, D).permute(0, 2, 3, 1, 4).reshape(B, H, -1, D), k.transpose(-1, -2).contiguous()) * SCALE
    del k
    scores = scores.view(B, H, Hq // H, T, L).masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-3e38))
    del scores
    total = p.sum(-1, keepdim=True)
    v = s["v_pages"][pages].float().transpose(1, 2).reshape(B, H, L, D).masked_fill(~seen.any(1)[:, None, :, None], 0.0)
    o = torch.matmul(p.view(B, H, -1, L), v).view(B, H, Hq // H, T, D)
    return torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(q.dtype)


def _plain_verify(s):
    x = s["logits"].double()
    B, T, V = x.shape
    b, i = torch.arange(B, device=DEVICE)[:, None], torch.arange(T, device=DEVICE)
    parents, tokens = s["parents"].long(), s["tokens"].long()
    there = _there(s, B, T)
    child = there & (parents >= 0) & (parents < i[None])
    of = torch.where(child, parents, 0)
    t = s["temperature"] if isinstance(s["temperature"], torch.Tensor) else torch.full((B,), s["temperature"], device=DEVICE)
    greedy = (t == 0)[:, None]
    first = lambda y: torch.where(y == y.amax(-1, keepdim=True), torch.arange(V, device=DEVICE), V).amin(-1)      # noqa: E731 (the lowest index of the largest)
    best = first(x)
    same = (of[:, :, None] == of[:, None, :]) & child[:, :, None] & child[:, None, :]
    earlier = same & (i[None, :] < i[:, None])
    passes = tokens == best[b, of]
    if s["noise"] is not None:
        x = x / torch.where(greedy, 1.0, t[:, None]).double()[:, :, None]
        p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
        if s["draft"] is None:
            repeated = (earlier & (tokens[:, :, None] == tokens[:, None, :])).any(-1)
            weight = torch.where(child & ~repeated, p[b, of, tokens], 0.0)
            left = p.sum(-1)[b, of] - (earlier * weight[:, None, :]).sum(-1)
            passes = torch.where(greedy, passes, s["accept"] * left < weight)
        else:
            p = p / p.sum(-1, keepdim=True)
            scale, less = torch.ones(B, T, dtype=torch.float64, device=DEVICE), torch.zeros(B, T, dtype=torch.float64, device=DEVICE)
            passes = torch.zeros_like(child)
            rank = earlier.sum(-1)
            q = s["draft"].double()
            for r in range(int(torch.where(child, rank + 1, 0).max())):      # the children of each node in turn, the rejected ones taken out
                now = child & (rank == r)
                px = (scale[b, of] * p[b, of, tokens] - less[b, of] * q[b, of, tokens]).clamp(min=0)
                passes |= now & (s["accept"] * q[b, of, tokens] < px)
                refused = torch.zeros(B, T, dtype=torch.int64, device=DEVICE).scatter_add_(1, of, (now & ~passes).long()) > 0
                less = torch.where(refused, less + 1, less)
                z = (scale[..., None] * p - less[..., None] * q).clamp(min=0).sum(-1)
                scale = torch.where(refused, torch.where(z > 0, scale / z, 1.0), scale)
                less = torch.where(refused, torch.where(z > 0, less / z, 0.0), less)
    passes = passes & child
    chosen = passes & ~(earlier & passes[:, None, :]).any(-1)
    ok = there & (chosen | (i[None] == 0))
    on_path = (ok[:, None, :] | ~_ancestors(parents)).all(-1)
    counts = on_path.sum(-1).int()
    path = torch.where(on_path, i[None], T).sort(-1).values
    last = torch.where(on_path, i[None], 0).amax(-1)
    row = b[:, 0]
    token = best[row, last]
    if s["noise"] is not None:
        if s["draft"] is None:
            away = torch.zeros(B, V, dtype=torch.int32, device=DEVICE).scatter_add_(1, tokens, (child & (of == last[:, None])).int()) > 0
            score = torch.where(away, -math.inf, x[row, last] + s["noise"])
        else:
            rest = (scale[row, last][:, None] * p[row, last] - less[row, last][:, None] * q[row, last]).clamp(min=0)
            score = torch.log(torch.where(rest.sum(-1, keepdim=True) > 0, rest, p[row, last])) + s["noise"]
        token = torch.where(greedy[:, 0], token, first(score))
    return {"path": torch.where(path < T, path, -1).int(), "counts": counts, "token": torch.where(counts > 0, token, -1)}


def _plain_move(s):
    R, page = s["rows"], s["k_pages"].size(3)
    i = torch.arange(R, device=DEVICE)
    starts = s["starts"].long()
    seq = torch.arange(starts.numel(), device=DEVICE)
    b, n = torch.nonzero(i[None] < s["counts"][:, None], as_tuple=True)
    to = starts[b] + n
    at = starts[b] + (n if s["index"] is None else s["index"].long()[b, n])
    source = seq[b] if s["sources"] is None else s["sources"].long()[b]
    from_page, to_page = s["table"].long()[source, at // page], s["table"].long()[b, to // page]
    for pages in (s["k_pages"], s["v_pages"]):
        pages[:, to_page, :, to % page] = pages[:, from_page, :, at % page]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "attend": _exact_attend, "verify": _exact_verify, "move": _exact_move}[s["kind"]](s)


def _exact_tree(s):
    parents, lens = s["parents"].tolist(), s["lens"].tolist()
    B, T = len(parents), len(parents[0])
    nodes = [T] * B if s["nodes"] is None else s["nodes"].tolist()
    mask, positions, slots = [], [], []
    for of, n, count in zip(parents, lens, nodes):
        lines = []
        for i in range(T):
            line = [i]
            while 0 <= of[line[-1]] < line[-1]:
                line.append(of[line[-1]])
            lines.append(line if i < count and n >= 0 else [])
        positions += [n + len(line) - 1 if line else -1 for line in lines]
        slots += [n + i if line else -1 for i, line in enumerate(lines)]
        mask.append([[sum(1 << j - 32 * w for j in line if j // 32 == w) for w in range(-(-T // 32))] for line in lines])
    mask = torch.tensor(mask, device=DEVICE)
    return {"mask": torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).int(), "positions": _ints(positions), "slots": _ints(slots)}


def _exact_attend(s):
    B, T, Hq, D = s["q"].shape
    H, size = s["k_pages"].shape[1:3]
    G = Hq // H
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=DEVICE)
    nodes = [T] * B if s["nodes"] is None else s["nodes"].tolist()
    masks = s["mask"].cpu().tolist()
    for b, n in enumerate(s["lens"].tolist()):
        if n < 0:
            continue
        m = nodes[b]
        first = max(0, n + 1 - s["window"]) if s["window"] else 0
        t = torch.arange(first, n + m, device=DEVICE)
        seen = torch.zeros(m, n + m, dtype=torch.bool)
        for i in range(m):
            of_tree = [n + j for j in range(m) if masks[b][i][j // 32] >> (j % 32) & 1]
            if s["window"] is None:
                seen[i, :n] = True
                seen[i, of_tree] = True
            else:
                last = (list(range(max(0, n - s["window"]), n)) + of_tree)[-s["window"]:]
                seen[i, last] = True
        away = ~seen[:, first:].to(DEVICE).repeat_interleave(G, 0)
        page = s["table"][b].long()[t // size]
        for h in range(H):
            keys, values = s["k_pages"][page, h, t % size].double(), s["v_pages"][page, h, t % size].double()
            q = s["q"][b, :m, h * G:(h + 1) * G].double().reshape(m * G, D)
            logit = (q @ keys.T.contiguous() * SCALE).masked_fill(away, -math.inf)
            out[b, :m, h * G:(h + 1) * G] = (torch.softmax(logit, dim=1) @ values).view(m, G, D)
    return out


def _exact_verify(s):
    B, T, V = s["logits"].shape
    parents, tokens = s["parents"].tolist(), s["tokens"].tolist()
    nodes = [T] * B if s["nodes"] is None else s["nodes"].tolist()
    t = s["temperature"].tolist() if isinstance(s["temperature"], torch.Tensor) else [s["temperature"]] * B
    lowest = lambda y: int((y == y.max()).nonzero()[0])      # noqa: E731
    paths, result = [], []
    for b in range(B):
        path = [0] if nodes[b] > 0 else []
        token = -1
        while path and token < 0:
            u = path[-1]
            x = s["logits"][b, u].double()
            p = None if t[b] == 0 else torch.softmax(x / t[b], 0)
            whole, found = p, None
            for c in (j for j in range(u + 1, nodes[b]) if parents[b][j] == u):
                y = tokens[b][c]
                if t[b] == 0:
                    ok = y == lowest(x)
                elif s["draft"] is None:
                    ok = float(s["accept"][b, c]) < float(p[y])
                    if not ok:
                        p = p.clone()
                        p[y] = 0
                        p = p / p.sum()
                else:
                    q = s["draft"][b, u].double()
                    ok = float(s["accept"][b, c].double() * q[y]) < float(p[y])
                    if not ok:
                        rest = (p - q).clamp(min=0)
                        p = rest / rest.sum() if float(rest.sum()) > 0 else whole
                if ok:
                    found = c
                    break
            if found is not None:
                path.append(found)
            else:
                token = lowest(x) if t[b] == 0 else lowest(p.log() + s["noise"][b].double())
        paths.append(path + [-1] * (T - len(path)))
        result.append(token)
    return {"path": _ints(paths), "counts": _ints([sum(j >= 0 for j in path) for path in paths]), "token": torch.tensor(result, device=DEVICE)}


def _exact_move(s):
    out = {}
    page = s["k_pages"].size(3)
    table, starts, counts = s["table"].tolist(), s["starts"].tolist(), s["counts"].tolist()
    moves = []
    for b, n in enumerate(counts):
        for i in range(n):
            at, to = starts[b] + (i if s["index"] is None else int(s["index"][b, i])), starts[b] + i
            seq = b if s["sources"] is None else int(s["sources"][b])
            moves.append((table[seq][at // page] * page + at % page, table[b][to // page] * page + to % page))
    old, new = (torch.tensor(list(x), device=DEVICE) for x in zip(*moves))
    for name in ("k_pages", "v_pages"):
        L, pool, H, _, D = s[name].shape
        rows = s[name].transpose(2, 3).reshape(L, pool * page, H, D).clone()
        rows[:, new] = s[name].transpose(2, 3).reshape(L, pool * page, H, D)[:, old]
        out[name] = rows.view(L, pool, page, H, D).transpose(2, 3).double()
    return out
