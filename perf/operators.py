"""Three operators of a decode step over sequences of unequal length, as cases that can be timed and compared.

``append``  ``ops.paged_append``: a step's or a prompt's queries, keys and values are normalised, rotated at each token's own
            position and mixed with value embeddings; keys and values go into the pages of a paged cache
``attend``  ``ops.paged_attention``: one new token per sequence against the pages of its sequence
``logits``  ``ops.process_logits``: penalties for repeated tokens, biases and grammar masks on the logits of a batch

With ``own`` false ``run`` computes them in elementary torch operations in 32 bits, rounded once; with ``own`` true through the
package's entry points.  ``exact`` computes the same from the definitions in 64 bits.  Head counts, head widths, windows, vocabularies
and prompt lengths are those of the repository's configurations, tests and benchmark, or generic.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
SCALE = 0.12                 # the framework's softmax scale
EPS = 1.1920928955078125e-07
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
LARGEST_BYTES = 2.2e9


# ---------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # One token of one sequence, the 12-head layer of the generator: launches and latency are all there is.
        dict(name="append_step_b1", kind="append", seqs=1, tokens=1, prompt=False, Hq=12, H=12, D=128, page=64, max_len=8192, cache="float16",
             norm=True, ve=False, copies=False, pad=0),
        # A decode step of a batch in which some slots are free: those tokens are skipped.
        dict(name="append_step_b64", kind="append", seqs=64, tokens=64, prompt=False, Hq=16, H=16, D=128, page=16, max_len=8192, cache="bfloat16",
             norm=True, ve=True, copies=False, pad=7),
        # Seven prompts of unequal length packed behind one another, narrow heads, value embeddings; attention reads the contiguous copies.
        dict(name="append_prompts_6001", kind="append", seqs=7, tokens=6001, prompt=True, Hq=12, H=12, D=64, page=128, max_len=8192, cache="bfloat16",
             norm=True, ve=True, copies=True, pad=0),
        # A long batch of prompts with four query heads to a key head, rotated but not normalised.
        dict(name="append_prompts_65536", kind="append", seqs=16, tokens=65536, prompt=True, Hq=32, H=8, D=128, page=64, max_len=16384, cache="bfloat16",
             norm=False, ve=False, copies=False, pad=0),
        # The generator's regime: one sequence, 12 heads, a context of 8192, the generator's default cache type.
        dict(name="attend_b1_8192", kind="attend", B=1, Hq=12, H=12, D=128, page=64, min_len=8192, max_len=8192, window=0, cache="float16", empty=0),
        # A batch of chats of unequal length under a sliding window, free slots among them.
        dict(name="attend_b64_window_4096", kind="attend", B=64, Hq=16, H=16, D=128, page=16, min_len=1, max_len=8300, window=4096, cache="bfloat16", empty=3),
        # Many short sequences of narrow heads: neither bandwidth nor one long row, but many small pieces.
        dict(name="attend_b256_short", kind="attend", B=256, Hq=8, H=8, D=64, page=16, min_len=1, max_len=300, window=0, cache="bfloat16", empty=5),
        # Eight query heads to a key head over contexts of very different length: the work has to be split by what is there.
        dict(name="attend_shared_heads_b32", kind="attend", B=32, Hq=64, H=8, D=128, page=64, min_len=100, max_len=32768, window=0, cache="bfloat16", empty=0),
        # Two contexts as long as the rotary tables: reading the cache is all there is.
        dict(name="attend_b2_131072", kind="attend", B=2, Hq=16, H=16, D=128, page=128, min_len=131001, max_len=131072, window=0, cache="bfloat16", empty=0),
        # The generator's repetition penalty over its last 128 tokens, one row.
        dict(name="logits_b1", kind="logits", B=1, V=50304, logits="float32", T=128, decayed=True, bias=0, allowed=False, rows=False),
        # A batch of requests with settings of their own, a shared bias, a grammar's mask, an odd vocabulary.
        dict(name="logits_b64_grammar", kind="logits", B=64, V=50257, logits="float32", T=2000, decayed=False, bias=1, allowed=True, rows=True),
        # A large batch over a large vocabulary with long histories and a bias per request, bf16 logits.
        dict(name="logits_b256_131072", kind="logits", B=256, V=131072, logits="bfloat16", T=4096, decayed=False, bias=2, allowed=True, rows=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "logits", "logits"])
    D = rng.choice([64, 128, 128, 256])
    H = rng.choice([1, 2, 4, 8, 12, 16])
    Hq = H * rng.choice([1, 1, 1, 2, 4, 8, 16])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    cache = rng.choice(["bfloat16", "bfloat16", "float16"])
    if kind == "append":
        prompt = rng.random() < 0.6
        seqs = _log_int(rng, 1, 32) if prompt else _log_int(rng, 1, 512)
        tokens = max(seqs, _log_int(rng, 1, 65536)) if prompt else seqs
        ve = Hq == H and rng.random() < 0.4
        return dict(kind=kind, seqs=seqs, tokens=tokens, prompt=prompt, Hq=Hq, H=H, D=D, page=page, max_len=max(1024, tokens), cache=cache,
                    norm=rng.random() < 0.6, ve=ve, copies=prompt and rng.random() < 0.5, pad=rng.choice([0, 0, min(3, tokens - 1)]))
    if kind == "attend":
        B = _log_int(rng, 1, 512)
        max_len = _log_int(rng, 1, 131072)
        min_len = max(1, rng.choice([max_len, max_len // 2, max_len // 100]))
        window = rng.choice([0, 0, _log_int(rng, 1, max_len)])
        return dict(kind=kind, B=B, Hq=Hq, H=H, D=D, page=page, min_len=min_len, max_len=max_len, window=window, cache=cache,
                    empty=rng.choice([0, 0, B // 8]))
    T = rng.choice([0, _log_int(rng, 1, 32768), _log_int(rng, 1, 4096)])
    return dict(kind=kind, B=_log_int(rng, 1, 256), V=_log_int(rng, 300, 200000), logits=rng.choice(["float32", "bfloat16", "float16"]), T=T,
                decayed=rng.random() < 0.4, bias=rng.choice([0, 1, 2]), allowed=T == 0 or rng.random() < 0.5, rows=rng.random() < 0.5)


def draw(rng):
    """One more case of the ranges above; none costs more than the largest listed one."""
    while True:
        case = _draw_once(rng)
        if case["kind"] == "attend" and case["B"] * case["max_len"] * case["H"] * case["D"] * 4 > 1.2 * LARGEST_BYTES:
            continue
        if case["kind"] == "attend" and case["B"] * case["max_len"] * case["Hq"] > 3e8:      # the plain form's scores
            continue
        if case["kind"] == "append" and case["tokens"] * (case["Hq"] + 2 * case["H"]) * case["D"] * 4 > LARGEST_BYTES:
            continue
        if work(case)["bytes"] <= 0.9 * LARGEST_BYTES:
            return case


def _lengths(case):
    """Context lengths of an ``attend`` case (the same for every seed): spread over the range on a logarithmic scale, the longest among
    them, ``empty`` slots without a sequence."""
    rng = random.Random(case["B"] * 1000003 + case["max_len"])
    lens = [_log_int(rng, case["min_len"], case["max_len"]) for _ in range(case["B"])]
    lens[rng.randrange(case["B"])] = case["max_len"]
    for b in rng.sample(range(case["B"]), min(case["empty"], case["B"] - 1)):
        lens[b] = 0
    return lens


def _prompt_lengths(case):
    rng = random.Random(case["tokens"] * 31 + case["seqs"])
    cuts = sorted(rng.sample(range(1, case["tokens"]), case["seqs"] - 1)) if case["seqs"] > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]


def _visible(case):
    return [min(n, case["window"]) if case["window"] else n for n in _lengths(case)]


def work(case):
    if case["kind"] == "append":
        n, rows = case["tokens"], case["Hq"] + 2 * case["H"]
        elements = n * case["D"] * (2 * rows + (case["H"] if case["ve"] else 0) + (2 * case["H"] if case["copies"] else 0))
        return {"bytes": 2 * elements + n * case["D"] * 4 + 12 * n, "flops": 10 * n * rows * case["D"]}
    if case["kind"] == "attend":
        keys = sum(_visible(case))
        return {"bytes": 4 * keys * case["H"] * case["D"] + 4 * case["B"] * case["Hq"] * case["D"] + 4 * keys // case["page"] + 4 * case["B"],
                "flops": 4 * keys * case["Hq"] * case["D"]}
    B, V = case["B"], case["V"]
    size = 4 if case["logits"] == "float32" else 2
    return {"bytes": 2 * B * V * size + 8 * B * case["T"] + (B * V // 8 if case["allowed"] else 0) + 4 * V * (0, 1, B)[case["bias"]],
            "flops": 4 * B * V + 4 * B * case["T"]}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=dtype)


def _rotary(D, rows):
    """Rotation tables of the framework's shape: fp32 [rows, D/2], the upper half of the frequencies zero."""
    freq = torch.cat([(1 / 1024) ** torch.linspace(0, 1, D // 4), torch.zeros(D // 2 - D // 4)]).double()
    theta = torch.outer(torch.arange(rows).double(), freq).to(DEVICE)
    return theta.cos().float().contiguous(), theta.sin().float().contiguous()


def _page_table(live, width, g):
    """int32 [S, width] with pages of a shuffled pool at the entries that ``live`` names (ranges of entries, one per sequence),
    -1 elsewhere (pages given back behind a window, or not taken yet); and the pool's size."""
    count = [max(0, hi - lo) for lo, hi in live]
    total = sum(count)
    pool = total + 3
    pages = torch.randperm(pool, generator=g, device=DEVICE)[:total].to(torch.int32).cpu()
    table = torch.full((len(live), width), -1, dtype=torch.int32)
    at = 0
    for s, ((lo, _), n) in enumerate(zip(live, count)):
        table[s, lo:lo + n] = pages[at:at + n]
        at += n
    return table.to(DEVICE), pool


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["kind"] == "append":
        return _prepare_append(case, g, random.Random(seed))
    if case["kind"] == "attend":
        return _prepare_attend(case, g)
    return _prepare_logits(case, g)


def _prepare_append(case, g, rng):
    n, S, Hq, H, D, page = case["tokens"], case["seqs"], case["Hq"], case["H"], case["D"], case["page"]
    width = -(-case["max_len"] // page)
    if case["prompt"]:
        lens = _prompt_lengths(case)
        seq = [s for s, m in enumerate(lens) for _ in range(m)]
        pos = [t for m in lens for t in range(m)]
        live = [(0, -(-m // page)) for m in lens]
    else:                                # every sequence somewhere in its context, its earlier pages not needed here
        seq = list(range(n))
        pos = [rng.randrange(case["max_len"]) for _ in range(n)]
        live = [(p // page, p // page + 1) for p in pos]
    for i in range(n - case["pad"], n):  # tokens of free slots
        pos[i] = -1
    table, pool = _page_table(live, width, g)
    qkv = _randn(g, n, Hq + 2 * H, D)    # the projection's output: three views of one tensor
    cos, sin = _rotary(D, case["max_len"])
    cache = DTYPES[case["cache"]]
    s = dict(kind="append", q=qkv[:, :Hq], k=qkv[:, Hq:Hq + H], v=qkv[:, Hq + H:], cos=cos, sin=sin, table=table,
             pos=torch.tensor(pos, dtype=torch.int32, device=DEVICE), rows=torch.tensor(seq, dtype=torch.int32, device=DEVICE) if case["prompt"] else None,
             k_pages=_randn(g, pool, H, page, D, dtype=cache), v_pages=_randn(g, pool, H, page, D, dtype=cache), eps=EPS if case["norm"] else None,
             ve=None, gate=None, k_out=None, v_out=None)
    if case["ve"]:
        s["ve"], s["gate"] = _randn(g, n, H, D), torch.sigmoid(_randn(g, 1, dtype=torch.float32))
    if case["copies"]:
        s["k_out"], s["v_out"] = torch.zeros_like(s["k"]).contiguous(), torch.zeros_like(s["v"]).contiguous()
    return s


def _prepare_attend(case, g):
    lens, page = _lengths(case), case["page"]
    live = [((max(0, n - case["window"]) if case["window"] else 0) // page, -(-n // page)) for n in lens]
    table, pool = _page_table(live, -(-case["max_len"] // page), g)
    cache = DTYPES[case["cache"]]
    return dict(kind="attend", q=_randn(g, case["B"], case["Hq"], case["D"], dtype=cache), table=table, window=case["window"] or None,
                k_pages=_randn(g, pool, case["H"], page, case["D"], dtype=cache), v_pages=_randn(g, pool, case["H"], page, case["D"], dtype=cache),
                lens=torch.tensor(lens, dtype=torch.int32, device=DEVICE))


def _prepare_logits(case, g):
    B, V, T = case["B"], case["V"], case["T"]
    uniform = lambda *shape: torch.rand(*shape, generator=g, device=DEVICE)      # noqa: E731
    setting = lambda lo, hi: lo + (hi - lo) * uniform(B) if case["rows"] else lo + 0.5 * (hi - lo)      # noqa: E731
    s = dict(kind="logits", logits=_randn(g, B, V, dtype=torch.float32).mul_(4).to(DTYPES[case["logits"]]), history=None, lens=None,
             repetition=1.0, presence=0.0, frequency=0.0, half_life=None, cap=None, bias=None, allowed=None)
    if T:
        # few tokens often, many tokens seldom; histories of unequal length, what lies behind one is not part of it
        s["history"] = (uniform(B, T).pow(3) * V).long().clamp_(max=V - 1)
        s["lens"] = (uniform(B) * T).int().clamp_(min=1) if B > 1 else torch.full((1,), T, dtype=torch.int32, device=DEVICE)
        s["repetition"] = setting(1.0, 1.3)
        if case["decayed"]:
            s["half_life"], s["cap"] = 140.0, 3.0
        else:
            s["cap"] = 1.0
            s["presence"], s["frequency"] = setting(0.0, 0.5), setting(0.0, 0.25)
    if case["bias"]:
        s["bias"] = _randn(g, *((V,) if case["bias"] == 1 else (B, V)), dtype=torch.float32)
    if case["allowed"]:
        words = torch.randint(-2 ** 31, 2 ** 31, (2, B, -(-V // 32)), generator=g, device=DEVICE).int()
        s["allowed"] = words[0] & words[1]
        if B > 4:
            s["allowed"][B // 2] = 0                  # a grammar that has come to an end
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(state):
    if state["kind"] == "append":
        return _own_append(state) if own else _plain_append(state)
    if state["kind"] == "attend":
        return _own_attend(state) if own else _plain_attend(state)
    return _own_logits(state) if own else _plain_logits(state)


def _own_append(s):
    from daisy_amd import ops
    q = ops.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["pos"], rows=s["rows"], q=s["q"], cos=s["cos"], sin=s["sin"],
                         eps=s["eps"], ve=s["ve"], gate=s["gate"], k_out=s["k_out"], v_out=s["v_out"])
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"], "k": s["k_out"], "v": s["v_out"]}


def _own_attend(s):
    from daisy_amd import ops
    return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], window=s["window"], scale=SCALE)


def _own_logits(s):
    from daisy_amd import ops
    return ops.process_logits(s["logits"], s["history"], s["lens"], repetition=s["repetition"], half_life=s["half_life"], cap=s["cap"],
                              presence=s["presence"], frequency=s["frequency"], bias=s["bias"], allowed=s["allowed"])


def _plain_append(s):
    q, k, v = (s[x].float() for x in "qkv")
    if s["eps"] is not None:
        q, k, v = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s["eps"]) for x in (q, k, v))
    there = s["pos"] >= 0
    pos = s["pos"].clamp(min=0).long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def rotated(x):
        x1, x2 = x.chunk(2, dim=-1)
        return torch.cat((x1 * cos + x2 * sin, x2 * cos - x1 * sin), dim=-1)

    q, k = rotated(q), rotated(k)
    if s["ve"] is not None:
        v = s["gate"] * v + (1 - s["gate"]) * s["ve"].float()
    seq = s["rows"].long() if s["rows"] is not None else torch.arange(pos.numel(), device=DEVICE)
    size = s["k_pages"].size(2)
    at = torch.nonzero(there)[:, 0]
    page, slot = s["table"][seq[at], pos[at] // size].long(), (pos % size)[at]
    cache = s["k_pages"].dtype
    s["k_pages"][page, :, slot] = k[at].to(cache)
    s["v_pages"][page, :, slot] = v[at].to(cache)
    if s["k_out"] is not None:
        s["k_out"][at] = k[at].to(s["k"].dtype)
        s["v_out"][at] = v[at].to(s["v"].dtype)
    return {"q": torch.where(there[:, None, None], q, 0.0).to(cache), "k_pages": s["k_pages"], "v_pages": s["v_pages"], "k": s["k_out"], "v": s["v_out"]}


def _plain_attend(s):
    q, table, lens = s["q"], s["table"], s["lens"]
    B, Hq, D = q.shape
    H, page = s["k_pages"].shape[1:3]
    L = table.size(1) * page
    pages = table.clamp(min=0).long()
    t = torch.arange(L, device=DEVICE)
    seen = t[None] < lens[:, None]
    if s["window"]:
        seen = seen & (t[None] >= lens[:, None] - s["window"])
    k = s["k_pages"][pages].float().transpose(1, 2).reshape(B, H, L, D)
    scores = torch.matmul(q.float().reshape(B, H, Hq // H, D), k.transpose(-1, -2)) * SCALE
    del k
    seen = seen[:, None, None]
    top = scores.masked_fill(~seen, -math.inf).amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.where(seen, torch.exp(scores - top), 0.0)
    total = p.sum(-1, keepdim=True)
    v = s["v_pages"][pages].float().transpose(1, 2).reshape(B, H, L, D)
    o = torch.matmul(p, v.masked_fill(~seen[:, 0, :, :, None], 0.0))
    return torch.where(total > 0, o / total, 0.0).reshape(B, Hq, D).to(q.dtype)


def _plain_logits(s):
    x = s["logits"].float()
    B, V = x.shape
    column = lambda value: value[:, None] if isinstance(value, torch.Tensor) else value      # noqa: E731
    if s["history"] is not None:
        age = s["lens"][:, None] - torch.arange(s["history"].size(1), device=DEVICE)[None]      # 1: the last token
        seen = (age > 0).float()
        weight = seen * torch.exp2(-age.clamp(min=0) / s["half_life"]) if s["half_life"] is not None else seen
        count = torch.zeros_like(x).scatter_add_(1, s["history"], seen)
        power = torch.zeros_like(x).scatter_add_(1, s["history"], weight)
        if s["cap"] is not None:
            power = power.clamp(max=s["cap"])
        strength = torch.as_tensor(column(s["repetition"]), device=DEVICE, dtype=torch.float32)
        strength = torch.pow(strength, power)
        x = torch.where(x > 0, x / strength, x * strength)
        x = x - column(s["frequency"]) * count - column(s["presence"]) * (count > 0)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["allowed"] is not None:
        v = torch.arange(V, device=DEVICE)
        x = torch.where((s["allowed"][:, v >> 5] >> (v & 31)) & 1 != 0, x, -math.inf)
    return x.to(s["logits"].dtype)


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    if case["kind"] == "attend":
        return _exact_attend(s)
    return _exact_logits(s)


def _exact_append(s):
    half = s["q"].size(2) // 2
    live = s["pos"] >= 0
    angle = s["pos"].long() * live
    c, d = s["cos"].double()[angle].unsqueeze(1), s["sin"].double()[angle].unsqueeze(1)
    done = {}
    for name in "qkv":
        x = s[name].double()
        if s["eps"] is not None:
            x = x / (x.pow(2).sum(2, keepdim=True) / x.size(2) + s["eps"]).sqrt()
        if name == "v":
            if s["ve"] is not None:
                g = s["gate"].double()
                x = s["ve"].double() + g * (x - s["ve"].double())
        else:
            turned = torch.empty_like(x)
            turned[..., :half] = c * x[..., :half] + d * x[..., half:]
            turned[..., half:] = c * x[..., half:] - d * x[..., :half]
            x = turned
        done[name] = x
    pool, H, size, D = s["k_pages"].shape
    seq = s["rows"].long() if s["rows"] is not None else torch.arange(s["pos"].numel(), device=DEVICE)
    which = live.nonzero().flatten()
    flat = s["table"].long()[seq, angle.div(size, rounding_mode="floor")] * size + angle % size
    out = {"q": done["q"] * live.double().view(-1, 1, 1), "k": None, "v": None}
    for name in "kv":
        rows = s[name + "_pages"].double().transpose(1, 2).reshape(pool * size, H, D)
        rows.index_copy_(0, flat[which], done[name][which])
        out[name + "_pages"] = rows.view(pool, size, H, D).transpose(1, 2).contiguous()
        if s[name + "_out"] is not None:
            out[name] = done[name] * live.double().view(-1, 1, 1)
    return out


def _exact_attend(s):
    B, Hq, D = s["q"].shape
    H, size = s["k_pages"].shape[1:3]
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(s["lens"].tolist()):
        first = max(0, n - s["window"]) if s["window"] else 0
        if n == first:
            continue
        t = torch.arange(first, n, device=DEVICE)
        page = s["table"][b].long()[t // size]
        for h in range(H):
            keys, values = s["k_pages"][page, h, t % size].double(), s["v_pages"][page, h, t % size].double()
            group = slice(h * (Hq // H), (h + 1) * (Hq // H))
            logit = s["q"][b, group].double() @ keys.T.contiguous() * SCALE
            out[b, group] = torch.softmax(logit, dim=1) @ values
    return out


def _exact_logits(s):
    rows = []
    V = s["logits"].size(1)
    value = lambda name, b: float(s[name][b]) if isinstance(s[name], torch.Tensor) else s[name]      # noqa: E731
    bit = torch.arange(32, device=DEVICE)
    for b in range(s["logits"].size(0)):
        x = s["logits"][b].double()
        if s["history"] is not None:
            n = int(s["lens"][b])
            told = s["history"][b, :n]
            age = torch.arange(n, 0, -1, device=DEVICE).double()
            weights = 0.5 ** (age / s["half_life"]) if s["half_life"] is not None else torch.ones_like(age)
            n_seen = torch.bincount(told, minlength=V)
            power = torch.bincount(told, weights=weights, minlength=V)
            if s["cap"] is not None:
                power = power.clamp(max=s["cap"])
            factor = torch.exp(power * math.log(value("repetition", b)))
            x = torch.where(x > 0, x / factor, x * factor) - value("frequency", b) * n_seen - value("presence", b) * (n_seen > 0).double()
        if s["bias"] is not None:
            x = x + (s["bias"] if s["bias"].dim() == 1 else s["bias"][b]).double()
        if s["allowed"] is not None:
            bits = (s["allowed"][b].long()[:, None] >> bit) & 1
            x[bits.flatten()[:V] == 0] = -math.inf
        rows.append(x)
    return torch.stack(rows)
