"""Products in 8-bit integers (int8): codes and results bit by bit against the definition, which leaves nothing to the order of a
sum; the edges of the types, strides, streams, graphs; the integer MLP inside a step."""
import pytest
import torch

import rows8_reference as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _rand(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, device="cuda", generator=g) * torch.exp(torch.randn(*shape[:-1], 1, device="cuda", generator=g))
    return x.to(dtype)


def _same(a, b):
    """Equal bit by bit but for the sign of zero, NaN in the same places."""
    a, b = a.cpu(), b.cpu()
    assert a.dtype == b.dtype and a.shape == b.shape
    assert torch.equal(torch.isnan(a.float()), torch.isnan(b.float()))
    assert torch.equal(torch.nan_to_num(a.float(), nan=0.0, posinf=1e38, neginf=-1e38), torch.nan_to_num(b.float(), nan=0.0, posinf=1e38, neginf=-1e38))


@pytest.mark.parametrize("unsigned", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 17), (2, 3, 66), (5, 128), (33, 163), (7, 1025), (4, 4096), (2, 8200), (3, 20000), (70000, 5)])
def test_codes_and_scales(shape, dtype, unsigned):
    from npa_b200.int8 import dequantize_rows, quantize_rows
    x = _rand(*shape, dtype=dtype)
    x.reshape(-1, shape[-1])[0] = 0
    codes, scales = quantize_rows(x, unsigned=unsigned)
    want, want_scales = ref.quantized(x, unsigned)
    assert codes.dtype == (torch.uint8 if unsigned else torch.int8) and codes.shape == x.shape and scales.shape == x.shape[:-1]
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(codes.cpu().long(), want)
    for out in TYPES:
        _same(dequantize_rows(codes, scales, out), (want.float() * want_scales[..., None]).to(out))


@pytest.mark.parametrize("cols", [9, 64, 700, 5000])
def test_codes_at_the_borders(cols):
    """Values half way between two codes and the nearest numbers on both sides, extreme rows, rows that are not finite."""
    from npa_b200.int8 import dequantize_rows, quantize_rows
    g = torch.Generator().manual_seed(cols)
    rows = []
    for top in (127.0, 1.0, 3.7, 1e-30, 3e38, 1.3e-38, 1e-40, 1e-45):
        scale = max(float(torch.tensor(top, dtype=torch.float64) / 127), 2.0 ** -126)
        at = (torch.randint(-126, 126, (cols,), generator=g).double() + 0.5) * float(torch.tensor(scale).float())
        v = at.float()
        step = torch.randint(-1, 2, (cols,), generator=g)
        v = torch.where(step > 0, torch.nextafter(v, torch.tensor(float("inf"))), torch.where(step < 0, torch.nextafter(v, torch.tensor(-float("inf"))), v))
        v = v.clamp(-top, top)
        v[0] = top
        rows.append(v)
    for bad in (float("inf"), float("-inf"), float("nan")):
        v = torch.randn(cols, generator=g)
        v[cols // 2] = bad
        rows.append(v)
    rows.append(torch.zeros(cols))
    x = torch.stack(rows).cuda()
    for unsigned in (False, True):
        codes, scales = quantize_rows(x, unsigned=unsigned)
        want, want_scales = ref.quantized(x, unsigned)
        assert torch.equal(codes.cpu().long(), want)
        _same(scales, want_scales)
        assert torch.isnan(dequantize_rows(codes, scales)[-4:-1]).all()
    assert (scales > 0)[:-4].all()


SHAPES = [(1, 16, 8), (1, 4096, 256), (1, 1000, 1537), (2, 33, 40), (4, 7, 3), (5, 4096, 130), (8, 2048, 64), (13, 1000, 1537), (16, 512, 512), (17, 128, 100),
          (31, 163, 128), (64, 66, 18), (100, 1, 1), (127, 129, 257), (128, 128, 128), (129, 256, 300), (333, 2048, 520), (1000, 163, 128), (2500, 66, 128),
          (257, 4100, 129), (4096, 128, 35), (300, 65536, 20), (1, 65536, 9)]


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("variant", range(4))
def test_products(M, K, N, variant):
    from npa_b200.int8 import linear_int8, quantize_rows
    dtype = TYPES[(M + variant) % 3]
    x = _rand(M, K, seed=M, dtype=dtype)
    w, t = quantize_rows(_rand(N, K, seed=N))
    bias = _rand(1, N, seed=3).reshape(N).to(TYPES[(N + variant) % 3]) if variant in (1, 3) else None
    relu = variant >= 2
    codes, scales = ref.quantized(x)
    want = ref.linear(codes, scales, w, t, bias, relu, dtype)
    _same(linear_int8(x, w, t, bias=bias, relu=relu), want)
    out = TYPES[(M + N) % 3]
    q, s = quantize_rows(x, unsigned=variant % 2 == 1)
    codes, scales = ref.quantized(x, variant % 2 == 1)
    want = ref.linear(codes, scales, w, t, bias, relu, out)
    _same(linear_int8(q, w, t, bias=bias, relu=relu, x_scales=s, out_dtype=out), want)


@pytest.mark.parametrize("M", [1, 16, 40, 200])
@pytest.mark.parametrize("K", [65536, 4096])
def test_largest_sums(M, K):
    """Codes at the ends of their range: the sum reaches 2^31 - 65,536 x 383 and is exact."""
    from npa_b200.int8 import linear_int8
    x = torch.full((M, K), 255, dtype=torch.uint8, device="cuda")
    w = torch.full((9, K), 127, dtype=torch.int8, device="cuda")
    w[1] = -127
    w[2] = -128
    w[3, ::2] = 0
    one = torch.ones(M, device="cuda")
    out = linear_int8(x, w, torch.ones(9, device="cuda"), x_scales=one)
    _same(out, ref.linear(x, one, w, torch.ones(9)))
    xs = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    _same(linear_int8(xs, w, torch.ones(9, device="cuda"), x_scales=one), ref.linear(xs, one, w, torch.ones(9)))


@pytest.mark.parametrize("M", [1, 5, 200])
def test_strides_and_offsets(M):
    """Columns of wider tensors, rows that repeat, transposed and unaligned weights, batched shapes, pitches that no vector load fits."""
    from npa_b200.int8 import linear_int8, quantize_rows
    K, N = 80, 72
    wide = _rand(M, K + 11, seed=1)
    w, t = quantize_rows(_rand(N, K, seed=2))
    odd = torch.empty(N * 83 + 5, dtype=torch.int8, device="cuda")[5:].view(N, 83)[:, :K]
    odd.copy_(w)
    lying = w.t().contiguous().t()
    padded = torch.full((N, 96), 77, dtype=torch.int8, device="cuda")
    padded[:, :K] = w
    for x in (wide[:, 3:3 + K], wide[:, :K].t().contiguous().t(), wide[:1, :K].expand(M, K), wide[:, :K].to(torch.bfloat16)[:, :K]):
        codes, scales = ref.quantized(x)
        want = ref.linear(codes, scales, w, t, None, False, x.dtype)
        for weights in (w, odd, lying, padded[:, :K]):
            _same(linear_int8(x, weights, t), want)
        q, s = quantize_rows(x)
        loose = torch.full((M, K + 7), 99, dtype=torch.int8, device="cuda")
        loose[:, 1:1 + K] = q
        _same(linear_int8(loose[:, 1:1 + K], w, t, x_scales=s, out_dtype=x.dtype), want)
    cube = wide[:, :K].reshape(1, M, K).expand(2, M, K)
    codes, scales = ref.quantized(cube)
    _same(linear_int8(cube, w, t), ref.linear(codes, scales, w, t))
    assert linear_int8(wide[0, :K], w, t).shape == (N,)
    assert linear_int8(wide[:0, :K], w, t).shape == (0, N)
    assert linear_int8(wide[:, :K], w[:0], t[:0]).shape == (M, 0)


@pytest.mark.parametrize("M", [1, 9, 300])
def test_rows_do_not_depend_on_their_neighbours(M):
    """A row with an infinity gives NaN and leaves the others as they are; a row alone gives what it gives in a batch."""
    from npa_b200.int8 import linear_int8, quantize_rows
    x = _rand(M, 200, seed=5)
    w, t = quantize_rows(_rand(50, 200, seed=6))
    y = linear_int8(x, w, t)
    assert torch.equal(linear_int8(x[M // 2], w, t), y[M // 2])
    x[M // 2, 7] = float("inf")
    z = linear_int8(x, w, t, relu=True)
    assert torch.isnan(z[M // 2]).all()
    rest = torch.arange(M, device="cuda") != M // 2
    assert torch.equal(z[rest], y[rest].clamp_min(0))


def test_mlp_is_its_two_layers():
    from npa_b200.int8 import Int8MLP, linear_int8, mlp_int8, quantize_rows
    for rows, k, hidden, n, seed in [(1, 66, 128, 18, 0), (127, 5, 128, 1, 1), (2500, 66, 128, 18, 2), (1000, 163, 128, 35, 3), (513, 176, 128, 48, 4),
                                     (300, 64, 256, 40, 5), (33, 200, 96, 7, 6), (70001, 83, 128, 19, 7),
                                     (60001, 114, 128, 24, 8), (40000, 250, 128, 64, 9)]:
        z = _rand(rows, k, seed=seed)
        z[rows // 2] = 0
        w1, t1 = quantize_rows(_rand(hidden, k, seed=10 + seed))
        w2, t2 = quantize_rows(_rand(n, hidden, seed=20 + seed))
        b1 = _rand(1, hidden, seed=30 + seed).reshape(hidden)
        y = mlp_int8(z, w1, t1, b1, w2, t2)
        h = linear_int8(z, w1, t1, bias=b1, relu=True)
        q, s = quantize_rows(h, unsigned=True)
        _same(y, linear_int8(q, w2, t2, x_scales=s))
        off = torch.empty(rows * k + 1, device="cuda")[1:].view(rows, k)  # rows that start off 16 bytes take the two products
        off.copy_(z)
        _same(mlp_int8(off, w1, t1, b1, w2, t2), y)
        codes, scales = ref.quantized(z)
        hr = ref.linear(codes, scales, w1, t1, b1, True)
        codes, scales = ref.quantized(hr, True)
        _same(y, ref.linear(codes, scales, w2, t2))
        if rows > 2:
            z[1, 0] = float("nan")
            again = mlp_int8(z.view(rows, 1, k), w1, t1, b1, w2, t2).view(rows, n)
            assert torch.isnan(again[1]).all()
            rest = torch.arange(rows, device="cuda") != 1
            assert torch.equal(again[rest], y[rest])
    module = torch.nn.Sequential(torch.nn.Linear(66, 128), torch.nn.ReLU(), torch.nn.Linear(128, 18, bias=False)).cuda()
    quick = Int8MLP(module)
    z = _rand(2, 400, 66)
    copy = Int8MLP(torch.nn.Sequential(torch.nn.Linear(66, 128), torch.nn.ReLU(), torch.nn.Linear(128, 18, bias=False)).cuda())
    copy.load_state_dict(quick.state_dict())
    with torch.no_grad():
        assert torch.equal(quick(z), copy(z)) and torch.equal(quick(z), copy.cpu().cuda()(z))


def test_refusals_on_the_device():
    from npa_b200.int8 import Int8MLP, dequantize_rows, linear_int8, mlp_int8, quantize_rows
    x = _rand(4, 32)
    w, t = quantize_rows(_rand(8, 32))
    q, s = quantize_rows(x)
    bad = [(RuntimeError, "32 columns", lambda: linear_int8(x, w[:, :16], t)), (RuntimeError, "w_scales must have shape", lambda: linear_int8(x, w, t[:3])),
           (RuntimeError, "need x_scales", lambda: linear_int8(q, w, t)), (RuntimeError, "belong to rows of codes", lambda: linear_int8(x, w, t, x_scales=s)),
           (RuntimeError, "x_scales must have shape", lambda: linear_int8(q, w, t, x_scales=s[:2])), (RuntimeError, "bias must have shape", lambda: linear_int8(x, w, t, bias=t[:4])),
           (TypeError, "w: expected int8", lambda: linear_int8(x, w.float(), t)), (TypeError, "x: expected", lambda: linear_int8(x.double(), w, t)),
           (TypeError, "out_dtype", lambda: linear_int8(x, w, t, out_dtype=torch.float64)), (TypeError, "w_scales: expected float32", lambda: linear_int8(x, w, t.half())),
           (TypeError, "w: expected a tensor on", lambda: linear_int8(x, w.cpu(), t)), (TypeError, "bias: expected a tensor on", lambda: linear_int8(x, w, t, bias=t.cpu())),
           (RuntimeError, "at least one column", lambda: quantize_rows(x[:, :0])), (RuntimeError, "at least 1 dimension", lambda: quantize_rows(x[0, 0])),
           (TypeError, "codes: expected int8 or uint8", lambda: dequantize_rows(x, s)), (RuntimeError, "scales must have shape", lambda: dequantize_rows(q, s[:1])),
           (ValueError, "65536", lambda: linear_int8(x.new_zeros(1, 65537), w.new_zeros(8, 65537), t)),
           (RuntimeError, "no backward", lambda: linear_int8(x.clone().requires_grad_(True), w, t)), (RuntimeError, "no backward", lambda: quantize_rows(x.clone().requires_grad_(True))),
           (RuntimeError, "b1 must have shape", lambda: mlp_int8(x, w, t, t[:7], w, t)), (RuntimeError, "8 columns", lambda: mlp_int8(x, w, t, t, w, t)),
           (ValueError, "Sequential", lambda: Int8MLP(torch.nn.Linear(3, 4).cuda())), (ValueError, "Sequential", lambda: Int8MLP(torch.nn.Sequential(torch.nn.Linear(3, 4), torch.nn.Tanh(), torch.nn.Linear(4, 2)).cuda()))]
    for error, text, call in bad:
        with pytest.raises(error, match=text):
            call()
    with torch.no_grad():
        linear_int8(x.clone().requires_grad_(True), w, t)


@pytest.mark.parametrize("M", [1, 12, 700])
def test_other_streams_and_graphs(M):
    """Two streams at once, and a graph replayed on new inputs: every call has its own workspace."""
    from npa_b200.int8 import linear_int8, quantize_rows
    x = [_rand(M, 640, seed=k) for k in range(3)]
    w, t = quantize_rows(_rand(300, 640, seed=9))
    want = [linear_int8(v, w, t) for v in x]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for r in range(10):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append((k, linear_int8(x[k], w, t)))
    torch.cuda.synchronize()
    for k, y in got:
        assert torch.equal(y, want[k])
    held = [x[0].clone(), x[1].clone()]
    graphs = []
    for v in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = linear_int8(v, w, t)
        graphs.append((g, y))
    held[0].copy_(x[2])
    held[1].copy_(x[0])
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want[2]) and torch.equal(graphs[1][1], want[0])


def test_a_step_with_an_integer_mlp():
    """step_euler runs an Int8MLP in evaluation: the update is that of its output."""
    from npa_b200 import sphops as sph
    from npa_b200.int8 import Int8MLP, mlp_int8
    from npa_b200.stepping import perceive, step_euler

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.model = torch.nn.Sequential(torch.nn.Linear(66, 128), torch.nn.ReLU(), torch.nn.Linear(128, 18, bias=False))
            self.eps0, self.alpha, self.spatial_dims = 0.1, 0.5, 2

    torch.manual_seed(0)
    model = Model().cuda()
    model.model = Int8MLP(model.model)
    grid = sph.HashGrid(dim=2, boundary="clamped", mode="grid", grid_size=(16, 16), eps=0.1, num_particles=2500, batch_size=1)
    x, s = torch.rand(1, 2500, 2, device="cuda") - 0.5, torch.randn(1, 2500, 16, device="cuda")
    with torch.no_grad():
        z, x_bin, s_bin, snap = perceive(model, x, s, grid)
        m = model.model
        y = mlp_int8(z, m.w1, m.w1_scales, m.b1, m.w2, m.w2_scales)
        want = sph.step_update(y, x_bin, s_bin, snap, 0.5, 1.0, None, False)
        got = step_euler(model, x, s, grid, update_prob=1.0)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for _ in range(3):
            x, s, _ = step_euler(model, x, s, grid)
        assert torch.isfinite(x).all() and torch.isfinite(s).all()
    with pytest.raises(RuntimeError, match="no backward"):
        step_euler(model, x, s.requires_grad_(True), grid)


def test_first_call_inside_a_capture_and_traces():
    """A shape that no call has used before is recorded in a graph; torch.jit.trace keeps the operators as nodes."""
    from npa_b200.int8 import Int8MLP, linear_int8, quantize_rows
    x, z = _rand(190, 48, seed=1), _rand(77, 40, seed=2)
    w, t = quantize_rows(_rand(24, 48, seed=3))
    quick = Int8MLP(torch.nn.Sequential(torch.nn.Linear(40, 128), torch.nn.ReLU(), torch.nn.Linear(128, 9, bias=False)).cuda())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g), torch.no_grad():
        a, b = linear_int8(x, w, t, out_dtype=torch.float16), quick(z)
    g.replay()
    with torch.no_grad():
        assert torch.equal(a, linear_int8(x, w, t, out_dtype=torch.float16)) and torch.equal(b, quick(z))
        traced = torch.jit.trace(quick, z)
        other = _rand(77, 40, seed=9)
        assert torch.equal(traced(other), quick(other))


@pytest.mark.parametrize("shift", range(9))
def test_rows_of_every_alignment(shift):
    """Rows that start on 2, 4, 8 or 16 bytes, of lengths around the kernels' blocks."""
    from npa_b200.int8 import quantize_rows
    from npa_b200.rows8 import compress_rows
    for cols in (31, 64, 65, 127, 129, 192, 193, 255, 257, 511, 513, 1030, 4104, 8195):
        for dtype in TYPES:
            x = _rand(9, cols + 16, seed=cols, dtype=dtype)[:, shift:shift + cols]
            codes, scales = quantize_rows(x)
            want, want_scales = ref.quantized(x)
            assert torch.equal(codes.cpu().long(), want) and torch.equal(scales.cpu(), want_scales)
            assert torch.equal(compress_rows(x).restore(torch.float32).cpu(), ref.kept(x).float())


def test_more_columns_than_32_bits_count():
    """Refused before anything is read or allocated: the rows are one number repeated."""
    from npa_b200 import int8, rows8
    long = 2**32 + 32
    x, codes, one = (torch.zeros(1, 1, dtype=d, device="cuda") for d in (torch.float32, torch.int8, torch.float32))
    for call in (lambda: int8.quantize_rows(x.expand(1, long)), lambda: int8.dequantize_rows(codes.expand(1, long), one[0]),
                 lambda: int8.linear_int8(x.expand(1, long), codes.expand(1, long), one[0]), lambda: rows8.compress_rows(x.expand(1, long))):
        with pytest.raises(RuntimeError, match="columns"):
            call()
    with pytest.raises(RuntimeError, match="channels"):
        int8.linear_int8(x, codes.expand(long, 1), one[0].expand(long))
