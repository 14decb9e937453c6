"""Routing from given logits on the GPU against a plain implementation in 64 bits.

Whole numbers are equal.  A weight is computed in 64 bits on both sides and rounded once to f32: half a step, 2^-24 relative
(the two evaluations differ by a few 2^-53, which moves a rounding only next to a border: one step, 2^-23)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

SOFTMAX, SIGMOID = 0, 1


def plain(z, k, score, select_bias=None, logit_bias=None, norm=False, scale=1.0, G=1, kept=1):
    """Token by token: (idx, w, expert_rows, slot, row_token)."""
    z = z.double().cpu().numpy()
    T, E = z.shape
    with np.errstate(invalid="ignore", over="ignore"):
        if logit_bias is not None:
            z = z + logit_bias.double().cpu().numpy()
        idx, w = np.full((T, k), -1), np.zeros((T, k))
        for t in range(T):
            free = [e for e in range(E) if z[t, e] > -math.inf]
            if not free:
                continue
            if score == SOFTMAX:
                m = max(z[t, e] for e in free)
                p = {e: 1.0 if z[t, e] == m else math.exp(z[t, e] - m) for e in free}
                total = math.fsum(p.values())
                p = {e: v / total for e, v in p.items()}
            else:
                p = {e: float(1.0 / (1.0 + np.exp(-z[t, e]))) for e in free}
            c = {e: p[e] + (float(select_bias[e]) if select_bias is not None else 0.0) for e in free}
            if G > 1:
                gs = E // G
                marks = []
                for g in range(G):
                    two = sorted((c[e] for e in free if e // gs == g), reverse=True)[:2]
                    if two:
                        marks.append((-sum(two), g))
                groups = {g for _, g in sorted(marks)[:kept]}
                free = [e for e in free if e // gs in groups]
            best = sorted(free, key=lambda e: (-c[e], e))[:k]
            idx[t, : len(best)] = best
            w[t, : len(best)] = [p[e] for e in best]
    if norm:
        w = w / (w.sum(1, keepdims=True) + 1e-20)
    rows = np.bincount(idx[idx >= 0], minlength=E)
    pairs = sorted((idx[t, j], t, j) for t in range(T) for j in range(k) if idx[t, j] >= 0)
    slot, token = np.full((T, k), -1), np.full(T * k, -1)
    for r, (_, t, j) in enumerate(pairs):
        slot[t, j], token[r] = r, t
    return idx, w * np.float64(np.float32(scale)), rows, slot, token


def check(backend, z, k, score, **kw):
    names = dict(norm="norm_topk", scale="routed_scale", G="n_group", kept="topk_group")
    got = backend.route_logits_dev(z, k, score, **{names.get(n, n): v for n, v in kw.items()})
    want = plain(z, k, score, **kw)
    for name, g, v in zip(got._fields, got, want):
        if name != "w":
            assert np.array_equal(g.cpu().numpy(), v), name
    w = got.w.double().cpu().numpy()
    assert (np.abs(w - want[1]) <= 2.0**-23 * np.abs(want[1]) + 2.0**-149).all()
    return got


def logits(T, E, seed, dtype=torch.float32, spread=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn((T, E), device="cuda", generator=g) * spread).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 8), (1, 256, 8), (5, 33, 3), (31, 128, 32), (32, 512, 2), (33, 129, 8), (200, 64, 6), (1000, 384, 8)])
def test_sizes_and_types(gpu_backend, dtype, score, T, E, k):
    check(gpu_backend, logits(T, E, 1, dtype), k, score, norm=bool(T % 2), scale=2.5)


@pytest.mark.parametrize("T", [33, 64, 65, 97, 129, 256, 257, 512, 513, 1024, 1025, 4736, 4737, 9472, 9473, 18944, 18945])
def test_chunk_lines(gpu_backend, T):
    check(gpu_backend, logits(T, 16, 2), 2, SOFTMAX)


@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("E,G,kept,k", [(256, 8, 4, 8), (64, 32, 5, 8), (32, 32, 3, 3), (24, 3, 1, 8), (60, 4, 4, 5), (512, 2, 1, 4)])
def test_groups_and_bias(gpu_backend, score, E, G, kept, k):
    bias = logits(1, E, 3)[0] * 0.1
    check(gpu_backend, logits(70, E, 4), k, score, select_bias=bias, G=G, kept=kept, norm=True)
    check(gpu_backend, logits(70, E, 5), k, score, logit_bias=bias, G=G, kept=kept)


@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("G,kept", [(1, 1), (8, 3)])
def test_closed_experts_and_padded_tokens(gpu_backend, score, G, kept):
    z = logits(50, 64, 6)
    z[torch.rand((50, 64), device="cuda", generator=torch.Generator("cuda").manual_seed(7)) < 0.8] = -math.inf
    z[3], z[49] = -math.inf, math.nan
    z[5, 1:] = -math.inf                      # none left either: expert 0 was closed before
    z[6] = -math.inf
    z[6, [9, 17, 63]] = 0.0                   # one each in three groups
    z[7, ::2] = math.nan
    got = check(gpu_backend, z, 6, score, G=G, kept=kept, norm=True)
    assert (got.idx[[3, 49]] == -1).all() and (got.w[[3, 49]] == 0).all() and (got.idx[5] == -1).all()


def test_ties_infinities_and_lowest_values(gpu_backend):
    z = torch.zeros((8, 96), device="cuda")
    z[1, [90, 4, 33]] = math.inf
    z[2] = torch.finfo(torch.float32).min
    z[3, 7:] = torch.finfo(torch.float32).min
    z[4] = torch.arange(96, device="cuda") // 10
    z[5, 0], z[5, 1:] = 0.0, -0.0
    z[6, 50] = torch.finfo(torch.float32).max
    z[7] = -200.0                             # sigmoids below f32's range
    for score in (SOFTMAX, SIGMOID):
        check(gpu_backend, z, 8, score, norm=True)
        check(gpu_backend, z, 8, score, norm=True, G=4, kept=2)
    got = gpu_backend.route_logits_dev(z, 8, SOFTMAX)
    assert got.idx[0].tolist() == list(range(8)) and got.idx[1, :3].tolist() == [4, 33, 90]


@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
def test_biases_of_the_lowest_value(gpu_backend, score):
    # groups 0 and 1 are closed, 2 has one open expert, and two choices of group 3 leave f32 when added
    lowest = torch.finfo(torch.float32).min
    z = logits(6, 8, 8)
    z[:, :4] = -math.inf
    z[:, 5] = -math.inf
    bias = torch.zeros(8, device="cuda")
    bias[6:] = lowest
    check(gpu_backend, z, 2, score, select_bias=bias, G=4, kept=3)
    bias[6] = -math.inf  # (the plain form keeps what can be chosen alone)
    got = gpu_backend.route_logits_dev(z, 2, score, select_bias=bias, n_group=4, topk_group=3)
    assert (got.idx.cpu() == torch.tensor([4, 7])).all()
    bias[7], bias[4] = -math.inf, 1.0
    got = gpu_backend.route_logits_dev(z, 2, score, select_bias=bias, n_group=4, topk_group=3)
    assert (got.idx.cpu() == torch.tensor([4, -1])).all()


def test_scores_that_32_bits_do_not_tell_apart(gpu_backend):
    z = torch.full((1, 64), 20.0, device="cuda")
    z[0, 50], z[0, 13] = 20.00001, 20.000002  # sigmoids all 1 in f32
    assert check(gpu_backend, z, 3, SIGMOID).idx[0].tolist() == [50, 13, 0]


def test_strided_logits_and_given_results(gpu_backend):
    base = logits(40, 200, 8, torch.bfloat16)
    z = base[:, 5:101]
    want = gpu_backend.route_logits_dev(z.contiguous(), 4)
    out = [torch.full_like(t, 77) for t in want]
    got = gpu_backend.route_logits_dev(z, 4, out=out)
    for a, b, o in zip(got, want, out):
        assert torch.equal(a, b) and a is o


def test_no_tokens(gpu_backend):
    got = gpu_backend.route_logits_dev(torch.empty((0, 16), device="cuda"), 2)
    assert (got.expert_rows == 0).all() and got.idx.shape == (0, 2)


def test_calls_on_two_streams_and_in_graphs(gpu_backend):
    zs = [logits(3000, 128, 9 + i) for i in range(2)]
    want = [gpu_backend.route_logits_dev(z, 8, norm_topk=True) for z in zs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in zs], []
    for z, st in zip(zs, streams):
        with torch.cuda.stream(st):
            for _ in range(5):
                last = gpu_backend.route_logits_dev(z, 8, norm_topk=True)
        got.append(last)
        got.append(gpu_backend.route_logits_dev(z, 8, norm_topk=True, stream=st.cuda_stream))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(r, want[i // 2]))
    graphs, outs = [], []
    for z in zs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(gpu_backend.route_logits_dev(z, 8, norm_topk=True))
        graphs.append(g)
    for r in outs:
        for t in r:
            t.fill_(-5)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for r, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(r, w))


def test_refusals(gpu_backend):
    z = torch.zeros((4, 16), device="cuda")
    out = gpu_backend.route_logits_dev(z, 2)
    for bad in (lambda: gpu_backend.route_logits_dev(z.double(), 2), lambda: gpu_backend.route_logits_dev(z[0], 2), lambda: gpu_backend.route_logits_dev(z.cpu(), 2),
                lambda: gpu_backend.route_logits_dev(z.t(), 2), lambda: gpu_backend.route_logits_dev(z, 2, select_bias=torch.zeros(15, device="cuda")),
                lambda: gpu_backend.route_logits_dev(z, 2, logit_bias=torch.zeros(16)), lambda: gpu_backend.route_logits_dev(z, 3, out=out),
                lambda: gpu_backend.route_logits_dev(z, 2, out=out._replace(w=out.idx))):
        with pytest.raises(ValueError):
            bad()
    for kw in (dict(k=17), dict(k=0), dict(k=2, score=5), dict(k=2, n_group=3), dict(k=9, n_group=4, topk_group=2)):
        with pytest.raises(gpu_backend.CudaError):
            gpu_backend.route_logits_dev(z, **kw)
