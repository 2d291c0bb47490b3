"""What the functions for drafted trees and evictions take and refuse of tensors on the GPU, and their
calls side by side."""

import pytest
import torch

import paged_reference as ref
import trees_reference as trees
from exp3_amd import paged

pytestmark = pytest.mark.gpu

TOKENS = 3


def _call(four=False, seed=1):
    """A cache of small values, its page table, starts, a tree and a ledger."""
    gen = torch.Generator().manual_seed(seed)
    cache = paged.empty_pages(8, 16, 2, 128, "cuda", four_bit=four)
    for x in vars(cache).values():
        if x is not None:
            x.copy_(torch.randint(120, 124, x.shape, generator=gen) if x.dtype == torch.uint8
                    else torch.randn(x.shape, generator=gen))
    return dict(cache=cache, table=torch.arange(4, dtype=torch.int32, device="cuda")[None],
                starts=torch.full((1,), 5, dtype=torch.int32, device="cuda"),
                x=torch.randn(1, TOKENS, 2, 128, generator=gen).to(torch.bfloat16).cuda(),
                parents=torch.tensor([[-1, 0, 0]], dtype=torch.int32, device="cuda"),
                tokens=torch.tensor([[4, 7, 4]], device="cuda"),
                targets=torch.tensor([[4, 1, 2]], device="cuda"),
                masks=torch.tensor([[[1], [3], [5]]], device="cuda"),
                lse=torch.full((1, TOKENS, 2), 3.0, device="cuda"),
                weights=torch.rand(1, 2, 64, generator=gen).cuda(),
                positions=torch.full((1, 2, 64), -1, dtype=torch.int32, device="cuda"))


def _tree(z):
    return paged.tree_attention(z["x"], z["cache"], z["table"], z["starts"], z["masks"], 0.1)


def _accept(z):
    return paged.accept_drafts(z["cache"], z["table"], z["starts"], z["parents"], z["tokens"],
                               z["targets"])


def _keep(z):
    return paged.keep_path(z["cache"], z["table"], z["starts"], z["parents"])


def _gather(z):
    return paged.accumulate_weights(z["weights"], z["x"], z["lse"], z["cache"], z["table"], z["starts"],
                                    0.1)


def _evict(z):
    return paged.evict_tokens(z["cache"], z["table"], z["starts"], z["weights"], 4, z["positions"])


def _pages(z, change):
    return dict(z, cache=paged.PagedCache(change(z["cache"].key_pages), z["cache"].value_pages))


CALLS = (_tree, _accept, _keep, _gather, _evict)


@pytest.mark.parametrize("call", CALLS)
def test_pages_that_require_a_gradient_are_refused(gpu, call):
    z = _call()
    z["cache"].key_pages.requires_grad_()
    with pytest.raises(ValueError, match="requires a gradient"):
        call(z)
    with torch.no_grad():
        call(z)


@pytest.mark.parametrize("call,name", ((_tree, "x"), (_gather, "x"), (_gather, "lse"),
                                       (_gather, "weights"), (_evict, "weights")))
def test_tensors_that_require_a_gradient_are_refused(gpu, call, name):
    z = _call()
    z[name].requires_grad_()
    with pytest.raises(ValueError, match="requires a gradient"):
        call(z)
    with torch.no_grad():
        call(z)


def test_forward_tangents_are_refused(gpu):
    def dual(y):
        return torch.autograd.forward_ad.make_dual(y, torch.ones_like(y))

    z = _call()
    with torch.autograd.forward_ad.dual_level():
        for call in CALLS:
            with pytest.raises(ValueError, match="tangent"):
                call(_pages(z, dual))
        for call, name in ((_tree, "x"), (_gather, "x"), (_gather, "lse"), (_gather, "weights"),
                           (_evict, "weights")):
            with pytest.raises(ValueError, match="tangent"):
                call(dict(z, **{name: dual(z[name])}))


def test_traced_graphs_are_refused(gpu):
    from torch.fx.experimental.proxy_tensor import make_fx

    z = _call()
    for step, x in ((lambda y: _tree(dict(z, x=y)), z["x"]),
                    (lambda y: paged.draft_tree(y)[1], z["parents"]),
                    (lambda y: _accept(dict(z, targets=y))[0], z["targets"]),
                    (lambda y: _keep(dict(z, parents=y)), z["parents"]),
                    (lambda y: _gather(dict(z, lse=y)), z["lse"]),
                    (lambda y: _evict(dict(z, weights=y))[1], z["weights"])):
        with pytest.raises(ValueError, match="traced"):
            make_fx(step)(x)


def test_only_plain_tensors(gpu):
    """Lazily negated queries and LSEs are read with the sign, other such tensors refused."""
    z = _call()
    assert torch.equal(_tree(dict(z, x=torch._neg_view(-z["x"]))), _tree(z))
    sums = []
    for minus in (False, True):
        w = z["weights"].clone()
        _gather(dict(z, weights=w, lse=torch._neg_view(-z["lse"]) if minus else z["lse"]))
        sums.append(w)
    assert torch.equal(*sums) and not torch.equal(sums[0], z["weights"])
    for call, name in ((_gather, "weights"), (_evict, "weights"), (_tree, "masks"), (_accept, "tokens")):
        with pytest.raises(ValueError, match="plain"):
            call(dict(z, **{name: torch._neg_view(z[name])}))
    for call, name in ((_tree, "x"), (_gather, "lse")):
        zero = torch._efficientzerotensor(z[name].shape, dtype=z[name].dtype, device="cuda")
        with pytest.raises(ValueError, match="plain"):
            call(dict(z, **{name: zero}))


@pytest.mark.parametrize("four", (False, True))
def test_what_counts_as_written(gpu, four):
    z = _call(four)
    pages = [x for x in vars(z["cache"]).values() if x is not None]
    rest = [x for x in z.values() if isinstance(x, torch.Tensor)]

    def grown(call):
        before = [x._version for x in pages + rest]
        call()
        return [b._version > a for a, b in zip(before, pages + rest)]

    none = [False] * len(rest)
    assert grown(lambda: _tree(z)) == [False] * len(pages) + none
    assert grown(lambda: paged.draft_tree(z["parents"])) == [False] * len(pages) + none
    for call in (_accept, _keep, _evict):
        assert grown(lambda: call(z)) == [True] * len(pages) + none
    weights = [x is z["weights"] for x in rest]
    assert grown(lambda: _gather(z)) == [False] * len(pages) + weights
    ledger = [x is z["weights"] or x is z["positions"] for x in rest]
    assert grown(lambda: paged.evict_tokens(z["cache"], z["table"], z["starts"], z["weights"], 4,
                                            z["positions"], out=(z["weights"], z["positions"]))) == \
        [True] * len(pages) + ledger


def test_shapes_types_and_devices(gpu):
    z = _call()
    int32, long = z["parents"], z["tokens"]
    for call, more in (
            (_tree, dict(masks=z["masks"][:, :2])), (_tree, dict(masks=z["masks"].int())),
            (_tree, dict(masks=z["masks"].cpu())), (_tree, dict(x=z["x"].float())),
            (_tree, dict(x=z["x"][..., :64])), (_tree, dict(starts=z["starts"].long())),
            (_tree, dict(table=z["table"].cpu())), (_tree, dict(x=z["x"][0])),
            (_accept, dict(parents=long)), (_accept, dict(tokens=int32)),
            (_accept, dict(targets=long[:, :2])), (_accept, dict(targets=long.cpu())),
            (_accept, dict(cache=[])), (_accept, dict(cache=[z["cache"], z["cache"]])),
            (_accept, dict(cache=[z["cache"], _call(four=True)["cache"]])),
            (_accept, dict(cache=[z["cache"], paged.empty_pages(9, 16, 2, 128, "cuda")])),
            (_keep, dict(parents=long)), (_keep, dict(parents=int32[0])),
            (_gather, dict(weights=z["weights"][..., :63].contiguous())),
            (_gather, dict(weights=z["weights"].double())),
            (_gather, dict(weights=z["weights"].mT.contiguous().mT)),
            (_gather, dict(lse=z["lse"][:, :2])), (_gather, dict(lse=z["lse"].bfloat16())),
            (_gather, dict(lse=z["lse"].cpu())), (_gather, dict(x=z["x"][:, :, :1])),
            (_evict, dict(weights=z["weights"][:, :1].contiguous())),
            (_evict, dict(positions=z["positions"].long())),
            (_evict, dict(positions=torch.cat([z["positions"]] * 2, -1))),
            (_evict, dict(starts=z["starts"][None]))):
        with pytest.raises(ValueError):
            call(dict(z, **more))
    evict = (z["cache"], z["table"], z["starts"], z["weights"])
    for more in (dict(budget=0), dict(budget=-1), dict(budget=4, recent=5), dict(budget=4, sinks=5),
                 dict(budget=4, recent=3, sinks=2), dict(budget=4, recent=-1),
                 dict(budget=4, out=(z["weights"], None)), dict(budget=4, seen=z["starts"].long()),
                 dict(budget=4, out=(z["weights"], z["positions"].float()))):
        with pytest.raises(ValueError):
            paged.evict_tokens(*evict, **more)
    with pytest.raises(ValueError, match="rope"):
        paged.append_tokens(z["cache"], z["table"], z["starts"], z["x"], z["x"], positions=int32)
    rope = paged.rope_table(64, 128, device="cuda")
    for positions in (long, int32[:, :2], int32.cpu()):
        with pytest.raises(ValueError):
            paged.append_tokens(z["cache"], z["table"], z["starts"], z["x"], z["x"], rope=rope,
                                positions=positions)
    for parents in (int32[0], long, int32[:, :0], torch.zeros(1, 257, dtype=torch.int32, device="cuda"),
                    torch.zeros(3, 2, dtype=torch.int32, device="cuda").T):
        with pytest.raises(ValueError):
            paged.draft_tree(parents)
    with pytest.raises(ValueError, match="256"):
        _tree(dict(z, x=torch.zeros(1, 257, 2, 128, dtype=torch.bfloat16, device="cuda")))


def test_calls_of_nothing(gpu):
    """No sequences; no tokens."""
    z = _call()
    empty = {name: x[:0] for name, x in z.items() if isinstance(x, torch.Tensor)}
    empty["cache"] = z["cache"]
    before = z["cache"].key_pages.clone()
    assert _tree(empty).shape == (0, TOKENS, 2, 128)
    assert [x.shape[0] for x in _accept(empty)] == [0, 0, 0]
    assert _keep(empty) is None and _gather(empty) is None
    assert [x.shape[0] for x in _evict(empty)] == [0, 0, 0]
    assert [x.shape[0] for x in paged.draft_tree(z["parents"][:0])] == [0, 0]
    none = dict(z, x=z["x"][:, :0], masks=z["masks"][:, :0, :0], lse=z["lse"][:, :0],
                parents=z["parents"][:, :0])
    weights = z["weights"].clone()
    assert _tree(none).shape == (1, 0, 2, 128)
    assert _gather(none) is None and _keep(none) is None
    assert torch.equal(weights, z["weights"]) and torch.equal(before, z["cache"].key_pages)


@pytest.mark.parametrize("tokens", (1, 9, 200))
def test_weights_on_two_streams(gpu, tokens):
    """Calls at once on two streams, each with its own workspace, and the LSE of any strides."""
    calls, want = [], []
    for seed in (61, 62):
        s = ref.make(seed, 2, tokens, 28, 4, 128, 64, 60, (3500, 900))
        cache, table, starts, _ = ref.on_gpu(s)
        lse = torch.full((2, 28, tokens), 4.0, device="cuda").mT
        calls.append((s.q.cuda(), lse, cache, table, starts, 0.1))
        want.append(torch.zeros(2, 4, 3840, device="cuda"))
        paged.accumulate_weights(want[-1], *calls[-1])
        other = torch.zeros_like(want[-1])
        paged.accumulate_weights(other, calls[-1][0], lse.contiguous(), *calls[-1][2:])
        assert torch.equal(want[-1], other)
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[torch.zeros_like(want[0]) for _ in range(4)] for _ in calls]
    torch.cuda.synchronize()
    for i in range(4):
        for stream, call, sums in zip(streams, calls, got):
            with torch.cuda.stream(stream):
                paged.accumulate_weights(sums[i], *call)
    torch.cuda.synchronize()
    for sums, right in zip(got, want):
        assert all(torch.equal(x, right) for x in sums)


def test_evictions_on_two_streams(gpu):
    calls = []
    for seed in (63, 64):
        s = ref.make(seed, 2, 1, 28, 4, 128, 64, 60, (3500, 900))
        cache, table, _, _ = ref.on_gpu(s)
        gen = torch.Generator().manual_seed(seed)
        weights = torch.rand(2, 4, 3840, generator=gen).cuda()
        lengths = torch.tensor([3501, 901], dtype=torch.int32, device="cuda")
        calls.append((cache, table, lengths, weights, 700))
    copies = [(paged.PagedCache(c.key_pages.clone(), c.value_pages.clone()), *more) for c, *more in calls]
    want = [paged.evict_tokens(*call, recent=9) for call in calls]
    torch.cuda.synchronize()
    got = []
    for call in copies:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(paged.evict_tokens(*call, recent=9))
    torch.cuda.synchronize()
    for (a, *_), (b, *_), x, y in zip(calls, copies, want, got):
        assert all(torch.equal(p, q) for p, q in zip(x, y))
        assert torch.equal(a.key_pages, b.key_pages) and torch.equal(a.value_pages, b.value_pages)


@pytest.mark.parametrize("bits", (16, 4))
def test_pages_past_32_bits(gpu, bits):
    """The same step in the first pages of a cache and behind 2^32 elements of a larger one."""
    s = ref.make(81, 2, 20, 28, 4, 128, 16, 24, (340, 90), bits=bits)
    near, table, starts, _ = ref.on_gpu(s)
    far = 2 ** 32 // (16 * 4 * 128) + 100
    large = paged.empty_pages(far + s.pages, 16, 4, 128, "cuda", four_bit=bits == 4)
    for x, y in zip(vars(large).values(), vars(near).values()):
        if y is not None:
            x[far:] = y
    q, parents = s.q.cuda(), trees.random_parents(81, 2, 20).cuda()
    _, masks = paged.draft_tree(parents)
    drafts = torch.zeros(2, 20, dtype=torch.int64, device="cuda")
    got = []
    for cache, at in ((near, table), (large, table + far)):
        weights = torch.zeros(2, 4, 384, device="cuda")
        out, lse = paged.tree_attention(q, cache, at, starts, masks, 0.1, return_lse=True)
        paged.accumulate_weights(weights, q, lse, cache, at, starts, 0.1)
        paged.accumulate_weights(weights, q[:, :1], lse[:, :1], cache, at, starts, 0.1)
        accepted, path, _ = paged.accept_drafts(cache, at, starts, parents, drafts, drafts)
        got.append([out, lse, weights, accepted, path,
                    *paged.evict_tokens(cache, at, starts + accepted, weights, 80, recent=5)])
    assert accepted.min() > 1
    for x, y in zip(*got):
        assert torch.equal(x, y)
    for x, y in zip(vars(large).values(), vars(near).values()):
        assert y is None or torch.equal(x[far:], y)


def _captured(seed):
    """A captured step on inputs of its own -> (graph, its outputs, the eager ones, what it reads)."""
    s = ref.make(seed, 2, 20, 28, 4, 128, 32, 40, (1100, 300))
    cache, table, starts, _ = ref.on_gpu(s)
    q = s.q.cuda()
    parents = trees.random_parents(seed, 2, 20).cuda()
    gen = torch.Generator().manual_seed(seed)
    drafts, targets = (torch.randint(0, 3, (2, 20), generator=gen).cuda() for _ in range(2))
    weights = torch.zeros(2, 4, 1280, device="cuda")
    held = cache.key_pages.clone(), cache.value_pages.clone()

    def step():
        cache.key_pages.copy_(held[0])
        cache.value_pages.copy_(held[1])
        weights.zero_()
        _, masks = paged.draft_tree(parents)
        out, lse = paged.tree_attention(q, cache, table, starts, masks, 0.1, return_lse=True)
        paged.accumulate_weights(weights, q, lse, cache, table, starts, 0.1)
        return (out, weights, *paged.accept_drafts(cache, table, starts, parents, drafts, targets),
                cache.key_pages, cache.value_pages)

    want = [x.clone() for x in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    return graph, got, want, step


def test_two_graphs_of_one_step(gpu):
    """Two captured steps of a tree, its weights and its acceptance, replayed in turn: neither keeps
    anything in the other's workspaces."""
    graphs = [_captured(seed) for seed in (71, 72)]
    for _ in range(3):
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, got, want, _ in graphs:
            assert all(torch.equal(x, y) for x, y in zip(got, want))
