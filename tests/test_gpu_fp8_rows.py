"""8-bit rows on the GPU: the row quantiser, the product with a resident weight, the experts over sorted rows, against plain
implementations in 64 bits.

Tolerances.  The product: codes multiply exactly; with n = K products summed in f32 in any order the sum is off by at most
(n + 4) 2^-24 of the sum of magnitudes (4: the scale product, its use, and the joins), plus the rounding of the result, half
a step of its type."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
EPS = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def to_e4m3(v):
    """The nearest e4m3 value of each f64 value, ties to even, at most 448."""
    a = v.abs().clamp_max(448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0**-6))) - 3.0)
    return torch.copysign((torch.round(a / step) * step).clamp_max(448.0), v)


def quantised(x):
    """f64 rows -> (values of the codes, scales): the definition in 64 bits."""
    q, s = torch.empty_like(x), []
    for c in range(0, x.shape[1], 128):
        b = x[:, c : c + 128]
        a = b.nan_to_num(nan=0.0, posinf=torch.inf, neginf=-torch.inf).abs().amax(1)
        s.append(torch.where(a > 0, (a / 448.0).clamp_min(2.0**-126), 1.0))
        q[:, c : c + 128] = to_e4m3(b / s[-1][:, None])
    return q, torch.stack(s, 1)


def spread(s, K):
    return s.repeat_interleave(128, 1)[:, :K]


def weight(backend, O, K, seed):
    """(resident handle, its values in f64)."""
    from speedycolibri_b200.configs import FMT_FP8_B128

    g = torch.Generator("cuda").manual_seed(seed)
    w = torch.randn((O, K), device="cuda", generator=g) * 0.05 * torch.exp(torch.randn((O, 1), device="cuda", generator=g))
    codes, scales = backend.quantize_fp8_b128_dev(w)
    v = codes.view(E4M3).double() * spread(scales.double(), K).repeat_interleave(128, 0)[:O]
    return backend.CudaTensor.from_device(FMT_FP8_B128, codes, scales, 1.0, K, O), v


def rows(T, K, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn((T, K), device="cuda", generator=g) * torch.exp(torch.randn((1, K), device="cuda", generator=g))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 128), (3, 129), (7, 100), (33, 2048), (130, 1000)])
def test_quantiser(gpu_backend, dtype, T, K):
    x = rows(T, K, 1).to(dtype)
    codes, scales = gpu_backend.quantize_rows_fp8_dev(x)
    q, s = quantised(x.double())
    # one rounding of the quotient a / 448, and of a value half-way between two codes either code is nearest to 2^-23 of it
    assert (scales.double() - s).abs().le(2.0**-24 * s).all()
    got, v = codes.view(E4M3).double(), x.double() / spread(s, K)
    assert ((got - v).abs() <= (q - v).abs() + 2.0**-22 * v.abs()).all()


def test_quantiser_at_odd_strides_and_places(gpu_backend):
    base = rows(40, 333, 2).to(torch.bfloat16)
    x = base[:, 3:301]  # rows 333 elements apart, off the 16-byte grid
    want = gpu_backend.quantize_rows_fp8_dev(x.contiguous())
    buf = torch.full((40, 512), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((40, 5), -7.0, device="cuda")
    gpu_backend.quantize_rows_fp8_dev(x, out=(buf[:, 16:314], scales[:, 1:4]))
    assert torch.equal(buf[:, 16:314], want[0]) and torch.equal(scales[:, 1:4], want[1])
    # 298 columns end on 304: zeros up to there, nothing touched around
    assert (buf[:, 314:320] == 0).all() and (buf[:, 320:] == 0x55).all() and (buf[:, :16] == 0x55).all()
    assert (scales[:, 0] == -7.0).all() and (scales[:, 4] == -7.0).all()


def test_quantiser_gathers(gpu_backend):
    x = rows(9, 260, 3)
    take = torch.tensor([8, 0, 0, -1, 5, 9, 8, 2**31 - 1, -(2**31)], dtype=torch.int32, device="cuda")
    codes = torch.full((9, 272), 0x33, dtype=torch.uint8, device="cuda")[:, :260]
    scales = torch.full((9, 3), -1.0, device="cuda")
    gpu_backend.quantize_rows_fp8_dev(x, take, out=(codes, scales))
    want = gpu_backend.quantize_rows_fp8_dev(x)
    for r, t in enumerate(take.tolist()):
        if 0 <= t < 9:
            assert torch.equal(codes[r], want[0][t]) and torch.equal(scales[r], want[1][t])
        else:
            assert (codes[r] == 0x33).all() and (scales[r] == -1.0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("K", [8, 136, 1000, 1032, 2048])
def test_gathered_rows_of_whole_pieces(gpu_backend, dtype, K):
    x = rows(70, K, 4).to(dtype)
    take = torch.arange(500, dtype=torch.int32, device="cuda") * 37 % 73  # (some past the last row)
    codes = torch.full((500, (K + 15) // 16 * 16), 0x33, dtype=torch.uint8, device="cuda")[:, :K]
    scales = torch.full((500, (K + 127) // 128), -1.0, device="cuda")
    gpu_backend.quantize_rows_fp8_dev(x, take, out=(codes, scales))
    want = gpu_backend.quantize_rows_fp8_dev(x)
    some = take < 70
    at = take[some].long()
    assert torch.equal(codes[some], want[0][at]) and torch.equal(scales[some], want[1][at])
    assert (codes[~some] == 0x33).all() and (scales[~some] == -1.0).all()


def test_quantiser_of_special_values(gpu_backend):
    x = torch.zeros((5, 256), device="cuda")
    x[1, 3], x[1, 4], x[1, 200] = torch.nan, 2.0, 1.0
    x[2, 5], x[2, 6], x[2, 130] = torch.inf, 3.0, 1.0
    x[3, 0], x[3, 1] = 1e-45, -1e-40
    x[4, 7], x[4, 8] = 3.4028234e38, -1.0
    codes, scales = gpu_backend.quantize_rows_fp8_dev(x)
    v = codes.view(E4M3).float()
    assert (v[0] == 0).all() and (scales[0] == 1).all()
    assert v[1, 3].isnan() and v[1, 4] == 448 and v[1, 200] == 448 and scales[1, 0] == np.float32(2.0) / np.float32(448.0)
    assert scales[2, 0] == torch.inf and v[2, 5].isnan() and v[2, 6] == 0 and v[2, 130] == 448
    assert scales[3, 0] == 2.0**-126 and v[3, 0] == 0 and (v[3, 1].double() * 2.0**-126 + 1e-40).abs() <= 2.0**-136
    assert v[4, 7] == 448 and v[4, 8] == 0


def product_bound(q, s, w, want, dtype):
    a = q.view(E4M3).double().abs() * spread(s.double(), q.shape[1])
    return (q.shape[1] + 4) * 2.0**-24 * (a @ w.abs().t()) + EPS[dtype] * want.abs() + 2.0**-25


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,K,O", [(1, 1, 1), (1, 128, 128), (1, 1024, 2048), (2, 300, 257), (8, 4096, 130), (9, 300, 4500), (16, 2048, 5000),
                                   (7, 200, 80000), (31, 1000, 1111), (128, 256, 256),
                                   (129, 384, 512), (333, 1000, 1111), (700, 640, 1000), (3000, 256, 2048)])
def test_product(gpu_backend, dtype, T, K, O):
    w, wv = weight(gpu_backend, O, K, 5)
    q, s = gpu_backend.quantize_rows_fp8_dev(rows(T, K, 6))
    y = gpu_backend.matmul_fp8_dev(w, q, s, out_dtype=dtype)
    gpu_backend.fp8_check()
    want = (q.view(E4M3).double() * spread(s.double(), K)) @ wv.t()
    assert y.dtype == dtype and ((y.double() - want).abs() <= product_bound(q, s, wv, want, dtype)).all()
    assert torch.equal(y, gpu_backend.matmul_fp8_dev(w, q, s, out_dtype=dtype))


def test_product_at_odd_strides(gpu_backend):
    T, K, O = 45, 300, 200
    w, _ = weight(gpu_backend, O, K, 7)
    q, s = gpu_backend.quantize_rows_fp8_dev(rows(T, K, 8))
    want = gpu_backend.matmul_fp8_dev(w, q, s, out_dtype=torch.float32)
    buf = torch.full((T, 512), 0x7F, dtype=torch.uint8, device="cuda")  # NaN codes around the rows
    buf[:, 32 : 32 + K] = q
    y = torch.full((T, 333), 5.0, device="cuda")
    gpu_backend.matmul_fp8_dev(w, buf[:, 32 : 32 + K], s.contiguous(), out=y[:, 7 : 7 + O])
    assert torch.equal(y[:, 7 : 7 + O], want) and (y[:, :7] == 5).all() and (y[:, 7 + O :] == 5).all()


@pytest.mark.parametrize("T", [5, 40, 200])
def test_nan_and_infinity_reach_their_row_only(gpu_backend, T):
    x = rows(T, 256, 9)
    x[1, 200], x[3, 4] = torch.nan, -torch.inf
    w, _ = weight(gpu_backend, 300, 256, 10)
    y = gpu_backend.matmul_fp8_dev(w, *gpu_backend.quantize_rows_fp8_dev(x))
    assert y[[1, 3]].isnan().all() and y[0].isfinite().all() and y[2].isfinite().all() and y[4:].isfinite().all()


def test_no_rows(gpu_backend):
    w, _ = weight(gpu_backend, 64, 64, 11)
    q, s = gpu_backend.quantize_rows_fp8_dev(torch.empty((0, 64), device="cuda"))
    assert gpu_backend.matmul_fp8_dev(w, q, s).shape == (0, 64)
    q, s = gpu_backend.quantize_rows_fp8_dev(torch.empty((4, 64), device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"))
    assert q.shape == (0, 64)


def expert_layer(backend, E, H, I, rows_cap, seed=20):
    from speedycolibri_b200.configs import FMT_FP8_B128
    from speedycolibri_b200.moe import Config, Expert, Layer, MoeBlock

    w = [[weight(backend, o, k, seed + 3 * e + i) for i, (o, k) in enumerate([(I, H), (I, H), (H, I)])] for e in range(E)]
    layer = Layer(np.zeros((E, H), np.uint16), [Expert(*(t for t, _ in m)) for m in w])
    return MoeBlock(Config(H, E, 1, I, fmt=FMT_FP8_B128), layer, max(1, rows_cap)), [[v for _, v in m] for m in w]


def expert_rows(q, s, counts, values):
    """(result of every row, how far it may be off), f64.  h and its codes in 64 bits; a value of h that lies within the f32 error of
    gate, up and the activation from a border between two codes may take either: its code then differs by one step."""
    H = q.shape[1]
    x = q.view(E4M3).double() * spread(s.double(), H)
    out, tol, at = [], [], 0
    for n, (g, u, d) in zip(counts, values):
        r = x[at : at + n]
        at += n
        eg, eu = (H + 4) * 2.0**-24 * (r.abs() @ g.abs().t()), (H + 4) * 2.0**-24 * (r.abs() @ u.abs().t())
        zg, zu = r @ g.t(), r @ u.t()
        h = zg * torch.sigmoid(zg) * zu
        # |silu'| <= 1.1, |silu(z)| <= |z|; the fast exponential and division: 2^-20 relative in all
        eh = 1.1 * eg * zu.abs() + zg.abs() * eu + 1.1 * eg * eu + 2.0**-20 * h.abs()
        hq, hs = quantised(h)
        sc = spread(hs, h.shape[1])
        lo, hi = to_e4m3((h - eh) / sc * (1 - 2.0**-20)), to_e4m3((h + eh) / sc * (1 + 2.0**-20))
        lo, hi = torch.minimum(lo, to_e4m3((h - eh) / sc * (1 + 2.0**-20))), torch.maximum(hi, to_e4m3((h + eh) / sc * (1 - 2.0**-20)))
        step = torch.maximum((hq - lo).abs(), (hi - hq).abs()) * sc  # 0 away from the borders
        # the scale moves with the row's largest value
        move = spread(torch.stack([(eh[:, c : c + 128]).amax(1) / 448.0 for c in range(0, h.shape[1], 128)], 1) + 2.0**-23 * hs, h.shape[1])
        v = hq * sc
        e = step * 1.01 + hq.abs() * move + (h.shape[1] + 4) * 2.0**-24 * v.abs()
        y = v @ d.t()
        out.append(y)
        tol.append(e @ d.abs().t() + 2.0**-8 * y.abs() + 2.0**-30)
    return torch.cat(out), torch.cat(tol)


@pytest.mark.parametrize("E,H,I,counts", [
    (1, 8, 8, [1]), (4, 64, 32, [0, 3, 0, 2]), (3, 256, 136, [1, 1, 1]), (8, 1024, 256, [1] * 8), (5, 320, 192, [130, 0, 7, 257, 1]),
    (6, 520, 264, [128, 129, 127, 0, 1, 300]), (16, 512, 512, [40] * 16), (40, 128, 128, [3, 0] * 20),
    (64, 1024, 136, [1] * 60 + [17, 0, 9, 2]), (12, 264, 520, [6] * 12), (300, 136, 264, [0, 1, 5] * 100)])
def test_experts(gpu_backend, E, H, I, counts):
    R = sum(counts)
    block, values = expert_layer(gpu_backend, E, H, I, R)
    q, s = gpu_backend.quantize_rows_fp8_dev(rows(R, H, 30))
    seg = torch.tensor(counts, dtype=torch.int32, device="cuda")
    y = torch.empty((R, H), dtype=torch.bfloat16, device="cuda")
    block.experts_fp8_dev(q, s, seg, R, y)
    block.check()
    want, tol = expert_rows(q, s, counts, values)
    assert ((y.double() - want).abs() <= tol).all()
    again = torch.empty_like(y)
    block.experts_fp8_dev(q, s, seg, R, again)
    assert torch.equal(y, again)
    block.close()


@pytest.mark.parametrize("expected", [0, 1, 6, 10000])
def test_rows_behind_the_last_segment_stay(gpu_backend, expected):
    counts, H = [2, 0, 4], 256
    block, _ = expert_layer(gpu_backend, 3, H, 128, 300)
    q, s = gpu_backend.quantize_rows_fp8_dev(rows(300, H, 31))
    q[6:] = 0x7F  # rows that belong to nobody
    y = torch.full((300, H), 3.0, dtype=torch.bfloat16, device="cuda")
    block.experts_fp8_dev(q, s, torch.tensor(counts, dtype=torch.int32, device="cuda"), expected, y)
    block.check()
    assert y[:6].isfinite().all() and (y[6:] == 3.0).all()
    block.close()


@pytest.mark.parametrize("expected", [1, 20])
@pytest.mark.parametrize("counts", [[5, 100, 5], [-3, 8, 2**31 - 1], [2**31 - 1, 2**31 - 1, 1], [0, 0, 0]])
def test_counts_past_the_buffer_are_cut(gpu_backend, counts, expected):
    H, R = 128, 20
    block, _ = expert_layer(gpu_backend, 3, H, 64, R)
    q, s = gpu_backend.quantize_rows_fp8_dev(rows(R, H, 32))
    cut, left = [], R
    for n in counts:
        cut.append(min(max(n, 0), left))
        left -= cut[-1]
    y, want = (torch.full((R, H), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    block.experts_fp8_dev(q, s, torch.tensor(counts, dtype=torch.int32, device="cuda"), expected, y)
    block.experts_fp8_dev(q, s, torch.tensor(cut, dtype=torch.int32, device="cuda"), expected, want)
    block.check()
    assert torch.equal(y, want) and (y[R - left :] == 3.0).all()
    block.close()


def test_offsets_past_32_bits(gpu_backend):
    T, K, O = 270000, 8192, 24  # 2.2 GB of codes
    x = torch.empty((T, K), dtype=torch.bfloat16, device="cuda")
    x[:1000], x[-1000:] = rows(1000, K, 50), rows(1000, K, 51)
    x[1000:-1000] = 1.0
    w, _ = weight(gpu_backend, O, K, 52)
    q, s = gpu_backend.quantize_rows_fp8_dev(x)
    y = gpu_backend.matmul_fp8_dev(w, q, s, out_dtype=torch.float32)
    for cut in (slice(0, 1000), slice(T - 1000, T)):
        qc, sc = gpu_backend.quantize_rows_fp8_dev(x[cut])
        assert torch.equal(qc, q[cut]) and torch.equal(sc, s[cut])
        want = (qc.view(E4M3).double() * spread(sc.double(), K)) @ weight_values(w, O, K).t()
        assert ((y[cut].double() - want).abs() <= product_bound(qc, sc, weight_values(w, O, K), want, torch.float32)).all()


def weight_values(w, O, K):
    """A handle's values in f64, through its export."""
    q, s, _ = w.export()
    return torch.from_numpy(q).cuda().view(E4M3).double() * spread(torch.from_numpy(s).cuda().double(), K).repeat_interleave(128, 0)[:O]


@pytest.mark.parametrize("T", [3, 100])
def test_streams_and_graphs(gpu_backend, T):
    """Calls on several streams at once, and captured ones replayed on other inputs."""
    K, O = 700, 600
    w, _ = weight(gpu_backend, O, K, 60)
    xs = [rows(T, K, 61 + i).to(torch.bfloat16) for i in range(3)]
    want = [gpu_backend.matmul_fp8_dev(w, *gpu_backend.quantize_rows_fp8_dev(x)) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], []
    for x, st in zip(xs, streams):
        with torch.cuda.stream(st):
            for _ in range(4):
                y = gpu_backend.matmul_fp8_dev(w, *gpu_backend.quantize_rows_fp8_dev(x))
        got.append(y)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = xs[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = gpu_backend.matmul_fp8_dev(w, *gpu_backend.quantize_rows_fp8_dev(x))
    for i in (1, 2, 0):
        x.copy_(xs[i])
        g.replay()
        assert torch.equal(y, want[i])
    gpu_backend.fp8_check()


def test_two_handles_at_once(gpu_backend):
    """Each handle has its own workspace: their calls may overlap."""
    H, I, counts = 512, 256, [3, 0, 70, 1]
    R = sum(counts)
    made = [expert_layer(gpu_backend, 4, H, I, R, seed=70 + 20 * i) for i in range(2)]
    seg = torch.tensor(counts, dtype=torch.int32, device="cuda")
    q, s = gpu_backend.quantize_rows_fp8_dev(rows(R, H, 80))
    want = [torch.empty((R, H), dtype=torch.bfloat16, device="cuda") for _ in made]
    for (block, _), y in zip(made, want):
        block.experts_fp8_dev(q, s, seg, R, y)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    got = [torch.empty_like(y) for y in want]
    for _ in range(5):
        for (block, _), y, st in zip(made, got, streams):
            block.experts_fp8_dev(q, s, seg, R, y, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for block, _ in made:
        block.check()
        block.close()


def test_refusals(gpu_backend):
    b, cuda = gpu_backend, "cuda"
    w, _ = weight(b, 64, 128, 90)
    q, s = b.quantize_rows_fp8_dev(torch.ones((4, 128), device=cuda))
    x = torch.ones((4, 128), device=cuda)
    for bad in (lambda: b.quantize_rows_fp8_dev(x.double()), lambda: b.quantize_rows_fp8_dev(x[0]), lambda: b.quantize_rows_fp8_dev(x.t()),
                lambda: b.quantize_rows_fp8_dev(x.cpu()), lambda: b.quantize_rows_fp8_dev(x, torch.zeros(4, dtype=torch.int64, device=cuda)),
                lambda: b.quantize_rows_fp8_dev(x, torch.zeros(4, dtype=torch.int32)), lambda: b.quantize_rows_fp8_dev(x, out=(q[:3], s[:3])),
                lambda: b.quantize_rows_fp8_dev(x, out=(q, s.double())), lambda: b.quantize_rows_fp8_dev(x, out=(q[:, :64], s)),
                lambda: b.matmul_fp8_dev(w, q[:, :64], s), lambda: b.matmul_fp8_dev(w, q, s[:3]), lambda: b.matmul_fp8_dev(w, q.cpu(), s),
                lambda: b.matmul_fp8_dev(w, q, s, out=torch.empty((4, 63), device=cuda)), lambda: b.matmul_fp8_dev(w, q, s, out_dtype=torch.float64),
                lambda: b.matmul_fp8_dev(w, q, s, out=torch.empty((64, 4), device=cuda).t()),
                lambda: b.matmul_fp8_dev(w, q, s, out_dtype=torch.float16, out=torch.empty((4, 64), device=cuda))):
        with pytest.raises(ValueError):
            bad()
    one = torch.zeros(128, dtype=torch.uint8, device=cuda)  # a row of 100 codes that ends with its storage's
    for part, fits in ((one[28:].view(1, 100), False), (one[16:116].view(1, 100), True)):
        if not fits:
            with pytest.raises(ValueError):
                b.quantize_rows_fp8_dev(x[:1, :100], out=(part, s[:1]))
        else:
            b.quantize_rows_fp8_dev(x[:1, :100], out=(part, s[:1]))
            assert (part == 0x7E).all() and (one[116:] == 0).all()  # 1 = 448 / 448, the largest code
    with pytest.raises(b.CudaError):  # rows of codes off the 16-byte grid
        b.matmul_fp8_dev(w, torch.zeros((4, 150), dtype=torch.uint8, device=cuda)[:, :128], s)
    block, _ = expert_layer(b, 2, 128, 64, 4)
    y, seg = torch.empty((4, 128), dtype=torch.bfloat16, device=cuda), torch.tensor([2, 2], dtype=torch.int32, device=cuda)
    for bad in (lambda: block.experts_fp8_dev(q, s, seg, 4, y.float()), lambda: block.experts_fp8_dev(q, s, seg[:1], 4, y),
                lambda: block.experts_fp8_dev(q, s, seg.long(), 4, y), lambda: block.experts_fp8_dev(q, s, seg.cpu(), 4, y),
                lambda: block.experts_fp8_dev(q, s, seg, 4, y[:3])):
        with pytest.raises(ValueError):
            bad()
    block.close()
