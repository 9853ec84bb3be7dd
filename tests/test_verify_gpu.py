"""``ops.verify_drafts`` against its definition, walked node by node in 64 bits: every number is an index, so all of it is compared exactly.

Where two numbers that decide are nearer to each other than the kernel's rounding (a sum of exponentials in fp32 pieces: 1e-6 of it; its products with
numbers below one, no more), the definition's walk says so, and the case takes other random numbers."""
import math
import random

import pytest
import torch

from daisy_amd import ops
from daisy_amd.generate import gumbel_noise
from test_paged_gpu import BF16, DEV, F16, gen
from test_tree_gpu import ints, random_parents

pytestmark = pytest.mark.gpu
F32 = torch.float32
NEAR = 1e-5


def walk(logits, tokens, parents, n, t, accept, noise, draft):
    """(path, token, nearest decision) of one sequence; everything on the CPU, in 64 bits."""
    path, gap = [0] if n > 0 else [], math.inf
    V = logits.shape[1]
    while path:
        u = path[-1]
        x = logits[u].double()
        if bool((x.isnan() | (x == math.inf)).any()) or bool((x == -math.inf).all()):
            return path, -1, gap
        kids = [c for c in range(u + 1, n) if parents[c] == u and 0 <= tokens[c] < V]
        found = None
        if not t > 0:
            best = int((x == x.max()).nonzero()[0])
            found = next((c for c in kids if tokens[c] == best), None)
            if found is None:
                return path, best, gap
            path.append(found)
            continue
        whole = torch.softmax(x / t, 0)
        p = whole.clone()
        gone = set()
        for c in kids:
            y = tokens[c]
            if draft is None:
                w, r = float(p[y]), float(p.sum())
                bar = float(accept[c].double()) * r
            else:
                w, bar = float(p[y]), float(accept[c].double() * draft[u, y].double())
            if w != bar:
                gap = min(gap, abs(w - bar) / max(w, bar))
            if bar < w:
                found = c
                break
            if draft is None:
                gone.add(y)
                p[y] = 0
            else:
                rest = (p - draft[u].double()).clamp(min=0)
                p = rest / rest.sum() if float(rest.sum()) > 0 else whole.clone()
        if found is not None:
            path.append(found)
            continue
        key = p.log() + noise.double()
        if not bool((key > -math.inf).any()):
            if draft is None:
                return path, -1, gap
            key = whole.log() + noise.double()
        top = key.topk(min(2, V)).values
        if V > 1:
            gap = min(gap, float(top[0] - top[1]))
        return path, int((key == key.max()).nonzero()[0]), gap
    return path, -1, gap


def check(s, what):
    t = s["temperature"]
    got = ops.verify_drafts(s["logits"], s["tokens"], s["parents"], nodes=s["nodes"], temperature=t, accept=s["accept"], noise=s["noise"], draft=s["draft"])
    path, counts, token = (x.cpu() for x in got)
    host = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    B, T, V = host["logits"].shape
    skipped = 0
    for b in range(B):
        n = T if host["nodes"] is None else min(max(int(host["nodes"][b]), 0), T)
        parents = host["parents"].tolist() if host["parents"].dim() == 1 else host["parents"][b].tolist()
        want, following, gap = walk(host["logits"][b], host["tokens"][b].tolist(), parents, n, float(t[b]) if isinstance(t, torch.Tensor) else t,
                                    None if host["accept"] is None else host["accept"][b], None if host["noise"] is None else host["noise"][b],
                                    None if host["draft"] is None else host["draft"][b])
        if gap < NEAR:
            skipped += 1
            continue
        assert path[b].tolist() == want + [-1] * (T - len(want)), f"{what}: sequence {b}: {path[b].tolist()}, {want}"
        assert counts[b] == len(want) and token[b] == following, f"{what}: sequence {b}: {token[b]}, {following}"
    assert skipped <= 1 + B // 20, f"{what}: {skipped} of {B} sequences decide by next to nothing"
    return got


def make(B, T, V, dtype=F32, shape="random", temperature=0.8, draft=False, kept=0, ragged=False, seed=0, few=None, int32=False):
    """``few``: drafted tokens from so many, so that children repeat each other's."""
    g, rng = gen(seed), random.Random(seed)
    parents = ints([random_parents(T, rng, shape) for _ in range(B)])
    logits = torch.randn(B, T, V, generator=g, device=DEV) * 3
    tokens = torch.randint(few or V, (B, T), generator=g, device=DEV)
    of = parents.clamp(min=0, max=T - 1).long()
    b = torch.arange(B, device=DEV)[:, None]
    q = None
    if draft:
        q = torch.softmax(logits + torch.randn(B, T, V, generator=g, device=DEV), -1)
        for i in range(1, T):
            tokens[:, i] = (q[b[:, 0], of[:, i]] / torch.empty(B, V, device=DEV).exponential_(generator=g)).argmax(-1)
    else:
        for i in range(1, T):
            logits[b[:, 0], of[:, i], tokens[:, i]] = 3 * math.sqrt(2 * math.log(V + 1)) + torch.randn(B, generator=g, device=DEV)
    if kept:
        logits = logits.masked_fill(logits < logits.topk(min(kept, V), -1).values[..., -1:], -math.inf)
    if temperature == "rows":
        temperature = torch.rand(B, generator=g, device=DEV) + 0.4
        temperature[::3] = 0.0
    u = torch.rand(B, V, generator=g, device=DEV).clamp_(min=1e-6)
    return dict(logits=logits.to(dtype), tokens=tokens.int() if int32 else tokens, parents=parents, nodes=ints([rng.randint(0, T) for _ in range(B)]) if ragged else None,
                temperature=temperature, accept=torch.rand(B, T, generator=g, device=DEV), noise=-torch.log(-torch.log(u)), draft=q)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [1, 2, 3, 255, 1000, 1023, 1024, 1025, 4099, 50257])
@pytest.mark.parametrize("temperature", [0.0, 0.8, "rows"])
def test_chosen_drafts_over_vocabularies(dtype, V, temperature):
    print(f"verify chosen {dtype} V{V} t{temperature}", flush=True)
    check(make(12, 7, V, dtype, temperature=temperature, seed=V), "chosen")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [1, 2, 3, 255, 1025, 4099, 50257])
@pytest.mark.parametrize("temperature,shape", [(1.0, "chain"), (0.7, "random"), ("rows", "star")])
def test_drawn_drafts_over_vocabularies(dtype, V, temperature, shape):
    print(f"verify drawn {dtype} V{V} t{temperature} {shape}", flush=True)
    check(make(12, 6, V, dtype, shape=shape, temperature=temperature, draft=True, seed=V + 1), "drawn")


@pytest.mark.parametrize("T", [1, 2, 31, 64, 65, 128, 200, 256])
@pytest.mark.parametrize("shape", ["chain", "random", "star", "forest"])
@pytest.mark.parametrize("draft", [False, True])
def test_trees_of_every_size(T, shape, draft):
    print(f"verify T{T} {shape} draft {draft}", flush=True)
    check(make(6, T, 700, shape=shape, draft=draft, ragged=True, seed=T), "trees")


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("B,T,V", [(1, 3, 200003), (300, 3, 500), (40, 16, 9000), (3, 40, 33000)])
def test_slices_and_rows_of_a_workgroup(B, T, V, draft):
    print(f"verify B{B} T{T} V{V} draft {draft}", flush=True)
    check(make(B, T, V, shape="random", draft=draft, temperature="rows", seed=B), "slices")


def test_children_with_the_same_token():
    for seed in range(4):
        check(make(20, 30, 400, shape="star", few=5, seed=seed, ragged=True), "repeats")
        check(make(20, 30, 400, shape="star", few=5, seed=seed, temperature=0.0), "repeats, greedy")


@pytest.mark.parametrize("kept", [1, 2, 20])
def test_filtered_rows(kept):
    """-inf for all but a few: often the children have all that is left."""
    for seed in range(4):
        check(make(30, 9, 1500, kept=kept, seed=seed), "kept")
        check(make(30, 9, 1500, kept=kept, seed=seed, temperature="rows"), "kept")


def test_masks_of_the_lowest_number_and_rows_of_nothing():
    for dtype in (F32, BF16, F16):
        s = make(9, 6, 900, dtype, seed=4, shape="chain")
        low = torch.finfo(dtype).min
        s["logits"][0] = torch.where(s["logits"][0] < 5, low, s["logits"][0])
        s["logits"][1, 0] = low                           # all alike: nothing but the noise decides
        s["logits"][2, 0] = -math.inf                     # nothing may follow
        s["logits"][3, 0] = -math.inf
        s["logits"][3, 0, int(s["tokens"][3, 1])] = 1.0   # the child alone may
        s["logits"][4, 0] = low
        s["logits"][4, 0, int(s["tokens"][4, 1])] = 3.0
        s["logits"][5, 1, 17] = float("nan")              # scores that are none: at the end of a path, or not on it
        s["logits"][6, 0, 899] = math.inf
        s["logits"][7, 5, 0] = float("nan")
        got = check(s, "lowest")
        assert got[2][2] == -1 and got[1][2] == 1 and got[0][3, 1] == 1 and got[0][4, 1] == 1 and got[2][6] == -1
        s["temperature"] = 0.0
        got = check(s, "lowest, greedy")
        assert got[2][2] == -1 and got[2][6] == -1


def test_draft_that_is_the_target_is_accepted_whole():
    s = make(16, 6, 3000, shape="chain", seed=5)
    s["temperature"] = 1.0
    s["draft"] = torch.softmax(s["logits"].double(), -1).float() * 0.999
    path, counts, _ = ops.verify_drafts(s["logits"], s["tokens"], s["parents"], temperature=1.0, accept=s["accept"], noise=s["noise"], draft=s["draft"])
    assert bool((counts == 6).all())


def test_draft_that_covers_the_target_leaves_the_target():
    """p <= q everywhere, a rejection leaves nothing: the draw is from p again, and so is the next child's test."""
    for shape in ("chain", "star"):
        s = make(16, 5, 800, shape=shape, seed=6, draft=True)
        s["draft"] = torch.softmax(s["logits"].double() / 0.8, -1).float() * 3
        s["accept"] = s["accept"] * 0.5 + 0.5
        check(s, "covered")


def test_tokens_outside_the_vocabulary_are_no_candidates():
    for draft in (False, True):
        s = make(8, 12, 300, seed=7, draft=draft)
        s["tokens"][:, 2], s["tokens"][:, 5], s["tokens"][:, 7] = -1, 300, 2 ** 40
        check(s, "outside")
        s["tokens"] = s["tokens"].clamp(-5, 400).int()
        check(s, "outside, int32")


def test_the_draw_is_the_targets():
    """What comes out behind the root, an accepted child or the token that follows, is distributed as p: chi squared over 12 tokens, 40000 draws."""
    B, V = 40000, 12
    g = gen(9)
    x = torch.randn(V, generator=g, device=DEV) * 1.5
    p = torch.softmax(x / 0.9, 0)
    for T, draft in ((1, False), (4, False), (3, True), (2, True)):
        logits = x.expand(B, T, V).contiguous()
        q = torch.softmax(x + torch.randn(V, generator=g, device=DEV), 0)
        tokens = torch.multinomial(q.expand(B, V), T, replacement=draft, generator=g)
        u = torch.rand(B, V, generator=g, device=DEV).clamp_(min=1e-6)
        path, counts, token = ops.verify_drafts(logits, tokens, ints([-1] + [0] * (T - 1)), temperature=0.9, accept=torch.rand(B, T, generator=g, device=DEV),
                                                noise=-torch.log(-torch.log(u)), draft=q.expand(B, T, V) if draft else None)
        first = torch.where(counts > 1, tokens.gather(1, path[:, min(1, T - 1)].clamp(min=0).long()[:, None])[:, 0], token)
        seen = torch.bincount(first, minlength=V).double()
        chi = ((seen - B * p.double()) ** 2 / (B * p.double())).sum().item()
        assert chi < 35, f"T{T} draft {draft}: {chi}"      # (11 degrees of freedom: above 35 once in 4000 times; the numbers are fixed)
        if T > 1:
            assert bool((counts > 1).any()) and bool((counts == 1).any())


def test_strides_shared_trees_and_workspaces():
    s = make(5, 6, 1001, BF16, seed=10, int32=True)
    want = check(s, "as it is")
    wide = torch.zeros(5, 9, 1010, dtype=BF16, device=DEV)
    wide[:, 2:8, 3:1004] = s["logits"]
    tokens = torch.zeros(5, 11, dtype=torch.int32, device=DEV)
    tokens[:, 4:10] = s["tokens"]
    noise = torch.zeros(5, 2000, device=DEV)
    noise[:, 1:1002] = s["noise"]
    accept = torch.zeros(5, 7, device=DEV)
    accept[:, 1:] = s["accept"]
    ws = torch.full((ops.verify_drafts_workspace_bytes(5, 6, 1001) + 64,), 255, dtype=torch.uint8, device=DEV)
    got = ops.verify_drafts(wide[:, 2:8, 3:1004], tokens[:, 4:10], s["parents"], temperature=0.8, accept=accept[:, 1:], noise=noise[:, 1:1002], workspace=ws)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    s["parents"] = s["parents"][2].contiguous()
    check(s, "one tree for all")
    s["noise"] = s["noise"][:1].expand(5, 1001)
    check(s, "one noise for all")


def test_replays_follow_their_inputs():
    s = make(4, 8, 5000, seed=11, ragged=True)
    call = lambda: ops.verify_drafts(s["logits"], s["tokens"], s["parents"], nodes=s["nodes"], temperature=0.8, accept=s["accept"], noise=s["noise"])      # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = call()
    for n in range(4):
        other = make(4, 8, 5000, seed=20 + n, ragged=True)
        for name in ("logits", "tokens", "parents", "nodes", "accept", "noise"):
            s[name].copy_(other[name])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(recorded, call())), n
    check(s, "the last one")


def test_generators_noise_serves():
    s = make(3, 4, 600, seed=12)
    s["noise"] = gumbel_noise(s["noise"])
    check(s, "noise")
