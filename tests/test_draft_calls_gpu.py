"""The operators of drafted trees called as programs call them: through the one-call path and the Python one, in views and lists of any strides, on other streams, twice at
once, and one behind the other in a recorded step."""
import pytest
import torch

from daisy_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Nothing:
    def __getattr__(self, name):
        return lambda *args: None


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def round_of(seed, B=3, T=9, H=2, G=2, D=64, page=16, V=101, dtype=torch.bfloat16, nodes=True):
    """Inputs of one step over trees, and the step: tree, append, attention, verification, moves."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens = ints([5, 0, 37][:B])
    pages = 5
    table = torch.randperm(B * pages, generator=g, device=DEV)[:B * pages].to(torch.int32).view(B, pages)
    half = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)      # noqa: E731
    s = dict(parents=ints([[-1] + [int(x) % max(i, 1) for i, x in enumerate(torch.randint(0, 100, (T - 1,), generator=g, device=DEV), 1)] for _ in range(B)]), lens=lens,
             nodes=ints([T, T - 4, 1][:B]) if nodes else None, table=table, k=half(2, B * pages, H, page, D), v=half(2, B * pages, H, page, D), q=half(B * T, H * G, D),
             new_k=half(B * T, H, D), new_v=half(B * T, H, D), logits=torch.randn(B, T, V, generator=g, device=DEV) * 3, tokens=torch.randint(0, V, (B, T), generator=g, device=DEV),
             accept=torch.rand(B, T, generator=g, device=DEV), noise=torch.randn(B, V, generator=g, device=DEV), status=torch.zeros(1, dtype=torch.int32, device=DEV))
    s["draft"] = torch.rand(B, T, V, generator=g, device=DEV).softmax(-1)
    return s


def run(s, temperature=1.0, draft=False, workspace=None):
    tree = ops.draft_tree(s["parents"], s["lens"], nodes=s["nodes"])
    B, T = s["tokens"].shape
    q = ops.paged_append(s["new_k"], s["new_v"], s["k"][0], s["v"][0], s["table"], tree.positions, rows=tree.rows, slots=tree.slots, q=s["q"], status=s["status"])
    o = ops.paged_tree_attention(q.view(B, T, *q.shape[1:]), s["k"][0], s["v"][0], s["table"], s["lens"], tree.mask, nodes=s["nodes"], window=20, status=s["status"], workspace=workspace)
    path, counts, following = ops.verify_drafts(s["logits"], s["tokens"], s["parents"], nodes=s["nodes"], temperature=temperature, accept=s["accept"], noise=s["noise"],
                                                draft=s["draft"] if draft else None)
    ops.paged_move(s["k"], s["v"], s["table"], s["lens"], counts, index=path, status=s["status"])
    return [*tree, q, o, path, counts, following, s["k"], s["v"], s["status"]]


def clone(s):
    return {k: None if v is None else v.clone() for k, v in s.items()}


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype,D,draft,nodes", [(torch.bfloat16, 64, False, True), (torch.float16, 128, True, True), (torch.bfloat16, 256, True, False)])
def test_both_paths_give_the_same(dtype, D, draft, nodes, monkeypatch):
    s = round_of(1, dtype=dtype, D=D, nodes=nodes)
    t = clone(s)
    one = run(s, draft=draft)
    with monkeypatch.context() as m:
        m.setattr(_lib, "native", lambda: Nothing())
        other = run(t, draft=draft)
    assert same(one, other) and s["status"].tolist() == [0]


def test_views_of_other_strides_and_integer_types():
    s = round_of(2)
    want = run(clone(s), temperature=torch.tensor([0.0, 0.7, 1.5], device=DEV))
    B, T, V = s["logits"].shape
    t = clone(s)
    t["logits"] = torch.randn(T, B, V + 7, device=DEV)
    t["logits"][..., 3:V + 3] = s["logits"].transpose(0, 1)
    t["logits"] = t["logits"][..., 3:V + 3].transpose(0, 1)
    for name, width in (("tokens", T + 3), ("parents", T + 3), ("accept", T + 2), ("noise", V + 5)):
        wide = torch.zeros(B, width, dtype=s[name].dtype, device=DEV)
        wide[:, 1:1 + s[name].shape[1]] = s[name]
        t[name] = wide[:, 1:1 + s[name].shape[1]]
    t["tokens"] = t["tokens"].int()
    for name in ("k", "v"):
        wide = torch.zeros(s[name].shape[1], 2, *s[name].shape[2:4], s[name].shape[4] + 8, device=DEV, dtype=s[name].dtype)
        wide[..., :s[name].shape[4]] = s[name].transpose(0, 1)
        t[name] = wide.transpose(0, 1)[..., :s[name].shape[4]]
    assert same(run(t, temperature=torch.tensor([0.0, 0.7, 1.5], device=DEV)), want)


def test_two_rounds_at_once_on_streams_of_their_own():
    rounds = [round_of(seed) for seed in (3, 4)]
    want = [run(clone(s), draft=True) for s in rounds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in rounds]
    for _ in range(5):
        mine = [clone(s) for s in rounds]
        torch.cuda.synchronize()
        got = []
        for stream, s in zip(streams, mine):
            with torch.cuda.stream(stream):
                got.append(run(s, draft=True))
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(got, want))


def test_two_recorded_rounds_replay_between_eager_ones():
    """Each recording has workspaces of its own; inputs change in place between the replays."""
    held, graphs, outs = [round_of(seed) for seed in (5, 6)], [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in held:
            run(clone(s))
    torch.cuda.current_stream().wait_stream(side)
    for s in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(s, draft=True))
        graphs.append(graph)
    for n in range(4):
        print(f"replay {n}", flush=True)
        for i, graph in enumerate(graphs):
            fresh = round_of(10 * n + i)
            for name, t in held[i].items():
                if t is not None:
                    t.copy_(fresh[name])
            want = run(clone(fresh), draft=True)
            graph.replay()
            torch.cuda.synchronize()
            assert same(outs[i], want), (n, i)


@pytest.mark.parametrize("B", [0, 1])
def test_no_sequences_and_one_node(B):
    s = round_of(7, B=max(B, 1), T=1, nodes=False)
    if B == 0:
        for name in ("parents", "lens", "table", "logits", "tokens", "accept", "noise", "draft"):
            s[name] = s[name][:0]
        tree = ops.draft_tree(s["parents"], s["lens"])
        assert tree.mask.shape == (0, 1, 1) and tree.rows.numel() == 0
        q = s["q"][:0].view(0, 1, 4, 64)
        assert ops.paged_tree_attention(q, s["k"][0], s["v"][0], s["table"], s["lens"], tree.mask).shape == (0, 1, 4, 64)
        path, counts, following = ops.verify_drafts(s["logits"], s["tokens"], s["parents"])
        assert path.shape == (0, 1) and counts.shape == following.shape == (0,)
        ops.paged_move(s["k"], s["v"], s["table"], s["lens"], counts, index=path)
        return
    out = run(s, temperature=0.0)
    assert out[-6].tolist() == [[0]] and out[-5].tolist() == [1] and out[-4].tolist() == [int(s["logits"][0, 0].argmax())]


def test_the_results_are_inference_tensors_nowhere():
    """Called under autograd with inputs that want no gradients, results want none."""
    out = run(round_of(8))
    assert not any(t.requires_grad for t in out)
