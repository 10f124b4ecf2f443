"""8-bit floating point in blocks of 128: the codes and scales against their definition, exactly; products against exact ones, where
every sum is a whole number that 32 bits hold, and against 64 bits; the layer with both gradients."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# The 8-bit matrix instruction adds 128 products cut off about 2^-17 below the largest: 128 * 2^-17 of a block's largest product at most.
CUT = 2.0 ** -10


def ops():
    from neural_block_textures_amd import ops as o
    return o


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(seed, *shape):
    return torch.randn(shape, generator=gen(seed), device="cuda")


def define(x, rows):
    """values (64 bits) and exponent bytes of x by the definition: E the smallest with amax <= 448 * 2^(E - 127), nearest even of four bits"""
    R, K = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -K % 128, 0, -R % rows)).view(-(-R // rows), rows, -1, 128)
    fin = torch.where(torch.isfinite(b), b.abs(), 0.0).amax(dim=(1, 3))
    mant, e = torch.frexp(fin)
    E = torch.where(fin > 0, e - 1 - 8 + 127 + (mant > 0.875).int(), 0).clamp_min(0)
    scale = torch.ldexp(torch.ones_like(fin, device="cpu"), (E - 127).cpu()).cuda()
    y = b / scale[:, None, :, None]
    _, ye = torch.frexp(y.abs().clamp_min(2.0 ** -6))
    unit = torch.ldexp(torch.ones_like(y, device="cpu"), (ye - 4).cpu()).cuda()
    q = torch.round(y / unit) * unit
    q = torch.where(torch.isfinite(b), q, math.nan)
    out = (q * scale[:, None, :, None]).view(-(-R // rows) * rows, -1)[:R, :K]
    return out, E


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), nan=1e300), torch.nan_to_num(b.double(), nan=1e300))


def holds(q, x, rows):
    want, E = define(x, rows)
    assert q.shape == tuple(x.shape) and q.block_rows == rows
    assert torch.equal(q.exps[:, :E.shape[1]].int(), E.int()), "scales"
    assert not q.exps[:, E.shape[1]:].any() and not q.codes[:, x.shape[1]:].any(), "padding"
    assert same(q.values(), want), "values"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,K", [(1, 1), (1, 128), (3, 127), (128, 128), (129, 129), (16, 512), (37, 1500), (300, 513), (513, 260)])
def test_quantize(R, K, dtype):
    print("quantize", R, K, dtype, flush=True)
    x = (randn(R + K, R, K) * torch.exp(3 * randn(1, R, 1)) * 3).to(dtype)
    x[R // 2, K // 2] = 0
    o = ops()
    for rows in (1, 128):
        q, t = o.fp8_quantize_both(x, rows)
        holds(q, x, rows)
        holds(t, x.t(), rows)
        for a, b in ((q, o.fp8_quantize(x, rows)), (t, o.fp8_quantize_t(x, rows))):
            assert torch.equal(a.codes, b.codes) and torch.equal(a.exps, b.exps)
    assert same(o.fp8_quantize(x, 128).values(), o.fp8_quantize_t(x, 128).values().t())


@pytest.mark.parametrize("dtypes", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (3, 300, 127), (129, 5, 513), (260, 390, 1000)])
def test_quantize_pair(M, N, K, dtypes):
    """Two matrices at once hold what each alone does."""
    import ctypes as C
    o = ops()
    x, w = randn(M, M, K).to(dtypes[0]), randn(N, N, K).to(dtypes[1])
    want = [*o.fp8_quantize_both(x, 1), *o.fp8_quantize_both(w, 128)]
    got = [o.Fp8Tensor(torch.full_like(q.codes, 77), torch.full_like(q.exps, 77), q.shape, q.block_rows) for q in want]
    descs = []
    for v, (q, t), rows in ((x, got[:2], 1), (w, got[2:], 128)):
        code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[v.dtype]
        descs.append(o.QuantizeDesc(v.data_ptr(), v.shape[0], K, K, code, rows, q.codes.data_ptr(), q.exps.data_ptr(), t.codes.data_ptr(), t.exps.data_ptr()))
    why = C.create_string_buffer(200)
    rc = o.library().ntc_op_fp8_quantize_pair(C.byref(descs[0]), C.byref(descs[1]), torch.cuda.current_stream().cuda_stream, why, 200)
    assert rc == 0, why.value
    for a, b in zip(got, want):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.exps, b.exps)


def test_quantize_at_the_ends():
    """Amax at and beside 448 scales, ties, subnormal codes, zeros, tiny and huge blocks, infinities and NaN."""
    x = torch.zeros(12, 256, device="cuda")
    x[0, :4] = torch.tensor([448.0, 449.0, 1.0, 2.0 ** -9], device="cuda")
    x[1, :4] = torch.tensor([448.0, -448.0, 17.0, 19.0], device="cuda")          # 17 and 19: ties between four-bit numbers
    x[2, :6] = torch.tensor([256.0, 2.0 ** -7, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 5 * 2.0 ** -10], device="cuda")
    x[3, 0] = 1e-38
    x[4, :3] = torch.tensor([3e38, 1.0, -3e38], device="cuda")
    x[5, :3] = torch.tensor([math.inf, 2.0, -math.inf], device="cuda")
    x[6, :3] = torch.tensor([math.nan, 2.0, 0.3], device="cuda")
    x[7, :] = math.inf
    x[8, :2] = torch.tensor([-0.0, 1e-45], device="cuda")
    x[9] = torch.linspace(-1, 1, 256, device="cuda")
    x[10] = 2.0 ** torch.linspace(-30, 10, 256, device="cuda")
    for rows in (1, 128):
        q, t = ops().fp8_quantize_both(x, rows)
        holds(q, x, rows)
        holds(t, x.t(), rows)


def test_quantize_strides():
    whole = randn(3, 70, 600)
    for x in (whole[:, 5:300], whole[::3, 1:257], whole.t()[10:200], whole[:1].expand(9, 600), whole.to(torch.bfloat16)[:, 3:131]):
        holds(ops().fp8_quantize(x), x, 1)
        holds(ops().fp8_quantize_t(x), x.t(), 1)


def whole_numbers(seed, R, K, rows):
    """small whole numbers times a power of two a block, so that every product and sum is exact"""
    x = torch.randint(-3, 4, (R, K), generator=gen(seed), device="cuda").float()
    e = torch.randint(0, 3, (-(-R // rows), -(-K // 128)), generator=gen(seed + 1), device="cuda").float()
    return x * (2.0 ** e).repeat_interleave(rows, 0)[:R].repeat_interleave(128, 1)[:, :K]


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 16, 128), (2, 64, 64), (5, 300, 200), (16, 256, 1024), (17, 33, 129), (64, 64, 640), (100, 130, 384), (128, 128, 128), (129, 257, 513),
                                   (256, 256, 256), (300, 700, 1100), (512, 260, 96), (1000, 512, 512), (7, 4097, 2000), (260, 250, 9000), (1, 5000, 700), (40, 48, 20000), (20, 9000, 300), (1500, 1500, 300), (3601, 3590, 520)])
@pytest.mark.parametrize("rows", [(1, 128), (1, 1), (128, 1)])
def test_products_of_whole_numbers_are_exact(M, N, K, rows):
    print("matmul", M, N, K, rows, flush=True)
    a, b = whole_numbers(M + K, M, K, rows[0]), whole_numbers(N + K, N, K, rows[1])
    qa, qb = ops().fp8_quantize(a, rows[0]), ops().fp8_quantize(b, rows[1])
    assert torch.equal(qa.values(), a) and torch.equal(qb.values(), b)
    want = a.double() @ b.double().t()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = ops().fp8_matmul(qa, qb, dtype)
        assert got.shape == (M, N) and torch.equal(got.double(), want.to(dtype).double()), dtype


def bound(a, b, want, dtype):
    """cut-off products of each block, 32-bit sums over the blocks, the result's rounding"""
    K = a.shape[1]
    pad = lambda x: torch.nn.functional.pad(x.double().abs(), (0, -K % 128)).view(x.shape[0], -1, 128)  # noqa: E731
    most = pad(a).amax(2) @ pad(b).amax(2).t()
    return CUT * most + 2.0 ** -20 * (pad(a).flatten(1) @ pad(b).flatten(1).t()) + want.abs() * HALF[dtype] * 1.01 + (2.0 ** -25 if dtype == torch.float16 else 0)


@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (3, 1000, 777), (33, 513, 2048), (200, 1030, 640), (700, 600, 1500), (512, 512, 4096), (64, 64, 65536)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_products_against_64_bits(M, N, K, dtype):
    print("matmul64", M, N, K, dtype, flush=True)
    qa, qb = ops().fp8_quantize(randn(1, M, K)), ops().fp8_quantize(randn(2, N, K) * 0.1, 128)
    a, b = qa.values(), qb.values()
    want = a.double() @ b.double().t()
    got = ops().fp8_matmul(qa, qb, dtype).double()
    assert ((got - want).abs() <= bound(a, b, want, dtype)).all()
    assert (got - want).norm() <= want.norm() * (4e-5 + HALF[dtype])       # 1.5e-5 measured for the instruction; the rounding's rms is below half a unit


def test_products_carry_nan_to_their_row_and_column_alone():
    x, w = randn(1, 70, 300), randn(2, 90, 300)
    x[3, 200], x[65, 5] = math.nan, math.inf
    w[80, 299] = -math.inf
    y = ops().fp8_matmul(ops().fp8_quantize(x), ops().fp8_quantize(w))
    bad = torch.isnan(y)
    assert bad[[3, 65]].all() and bad[:, 80].all()
    bad[[3, 65]] = False
    bad[:, 80] = False
    assert not bad.any()
    y = ops().fp8_linear(x[3:4].to(torch.bfloat16), ops().fp8_quantize(randn(2, 90, 300), 128))
    assert torch.isnan(y).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(1, 64, 128), (1, 1000, 1500), (2, 4096, 4096), (8, 77, 300), (15, 300, 129), (16, 256, 512), (17, 128, 1000), (32, 96, 8192), (33, 40, 640), (64, 500, 260), (70, 64, 100), (300, 200, 257)])
def test_inference_layer(M, N, K, dtype):
    """The layer on weights laid out once equals the product of the two quantized matrices, however few the rows."""
    print("layer", M, N, K, dtype, flush=True)
    x, w = (randn(M, M, K) * 3).to(dtype), ops().fp8_quantize(randn(N, N, K) * 0.05, 128)
    y = ops().fp8_linear(x, w)
    a, b = define(x, 1)[0], w.values()
    want = a @ b.double().t()
    assert y.dtype == dtype and ((y.double() - want).abs() <= bound(a, b, want, dtype)).all()
    wide = torch.zeros(M, K + 5, dtype=dtype, device="cuda")
    wide[:, 2:K + 2] = x
    assert torch.equal(ops().fp8_linear(wide[:, 2:K + 2], w), y)              # rows at a stride, off alignment
    assert torch.equal(ops().fp8_linear(x.view(1, M, 1, K), w), y.view(1, M, 1, N))


@pytest.mark.parametrize("rows", [1, 5, 16, 40])
def test_inference_rows_do_not_depend_on_the_others(rows):
    x, w = randn(1, 64, 700).to(torch.bfloat16), ops().fp8_quantize(randn(2, 300, 700), 128)
    x[rows:] = math.nan
    y = ops().fp8_linear(x[:rows], w)
    assert torch.isfinite(y).all()
    z = x.clone()
    z[rows:] = 0
    assert torch.equal(ops().fp8_linear(z[:rows], w), y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (5, 300, 100), (130, 129, 257), (512, 256, 128), (1003, 200, 90), (3000, 64, 64)])
def test_training_layer(M, N, K, dtype):
    print("train", M, N, K, dtype, flush=True)
    x, w, dy = (randn(1, M, K)).to(dtype), (randn(2, N, K) * 0.1).to(dtype), (randn(3, M, N) * 0.1).to(dtype)
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = ops().fp8_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    X, W, D = define(x.detach(), 1)[0], define(w.detach(), 128)[0], define(dy, 1)[0]
    Xt, Dt = define(x.detach().t(), 1)[0], define(dy.t(), 1)[0]
    for got, a, b in ((y, X, W), (dx, D, W.t()), (dw, Dt, Xt)):
        want = a @ b.t()
        assert got.dtype == dtype and got.shape == want.shape
        assert ((got.detach().double() - want).abs() <= bound(a, b, want, dtype)).all()


def test_training_layer_gradient_against_differences():
    """On values that 8 bits hold exactly the layer is the product itself, and its gradient that of differences of the product."""
    x, w = whole_numbers(1, 64, 128, 1).requires_grad_(True), whole_numbers(2, 32, 128, 128).requires_grad_(True)
    dy = torch.randint(-2, 3, (64, 32), generator=gen(3), device="cuda").float()
    dx, dw = torch.autograd.grad(ops().fp8_linear(x, w), (x, w), dy)
    f = lambda a, b: ((a @ b.t()) * dy.double()).sum()  # noqa: E731
    X, W = x.detach().double(), w.detach().double()
    for _ in range(4):
        u, v = (torch.randint(-3, 4, t.shape, generator=gen(9), device="cuda").double() for t in (X, W))
        assert f(X + u, W) - f(X - u, W) == 2 * (dx.double() * u).sum()         # linear in each: whole differences are exact
        assert f(X, W + v) - f(X, W - v) == 2 * (dw.double() * v).sum()


def test_one_sided_gradients_and_shapes():
    x, w = randn(1, 3, 7, 200).to(torch.bfloat16), randn(2, 50, 200).to(torch.bfloat16)
    for rx, rw in ((True, False), (False, True), (False, False)):
        a, b = x.clone().requires_grad_(rx), w.clone().requires_grad_(rw)
        y = ops().fp8_linear(a, b)
        assert y.shape == (3, 7, 50)
        if rx or rw:
            y.sum().backward()                          # a gradient of one number, expanded
            assert (a.grad is not None) == rx and (b.grad is not None) == rw
    e = ops().fp8_linear(torch.empty((0, 200), device="cuda"), w)
    assert e.shape == (0, 50)
    z = ops().fp8_linear(torch.empty((4, 0), device="cuda"), torch.empty((6, 0), device="cuda"))
    assert z.shape == (4, 6) and not z.any()


def test_other_streams_and_repeats():
    x, w = randn(1, 600, 1000).to(torch.bfloat16), randn(2, 500, 1000).to(torch.bfloat16)
    a, b = ops().fp8_quantize(x), ops().fp8_quantize(w, 128)
    long_a, long_b = ops().fp8_quantize_t(x), ops().fp8_quantize_t(w[:, :100].contiguous())
    want = [ops().fp8_matmul(a, b), ops().fp8_linear(x[:3], b), ops().fp8_matmul(long_a, ops().fp8_quantize_t(x), torch.float32)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            got = [ops().fp8_matmul(a, b), ops().fp8_linear(x[:3], b), ops().fp8_matmul(long_a, ops().fp8_quantize_t(x), torch.float32)]
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert long_b.shape == (100, 500)


def test_products_past_32_bit_offsets():
    print("matmul far rows", flush=True)
    M, K, N = 33000, 65536, 32                           # 2.16e9 codes in A
    codes = torch.zeros((M, K), dtype=torch.uint8, device="cuda")
    codes[0, :128] = 0x38                                # 1.0
    codes[-1] = 0x38
    a = ops().Fp8Tensor(codes, torch.full((M, K // 128), 127, dtype=torch.uint8, device="cuda"), (M, K), 1)
    b = ops().fp8_quantize(torch.ones((N, K), device="cuda"), 128)
    y = ops().fp8_matmul(a, b, torch.float32)
    assert (y[0] == 128).all() and (y[-1] == K).all() and not y[1:-1].any()


@pytest.mark.parametrize("rows", [1, 128])
def test_more_rows_than_a_grid_dimension_takes(rows):
    """A row's codes are its own block's, wherever it lies: the ends and the middle of 9 million rows as matrices of their own."""
    R, K, step = 9_000_001, 5, 128 * 2 ** 15
    print("quantize", R, K, rows, flush=True)
    x = randn(21, R, K).to(torch.bfloat16)
    q, t = ops().fp8_quantize_both(x, rows)
    for a in (0, step - 256, step, 2 * step - 128, 2 * step, R // 128 * 128):
        b = min(R, a + 512)
        one, other = ops().fp8_quantize_both(x[a:b], rows)
        assert torch.equal(q.codes[a:b], one.codes), a
        assert torch.equal(q.exps[a // rows:(b + rows - 1) // rows], one.exps), a
        assert torch.equal(t.codes[:, a:b], other.codes[:, :b - a]), a
        n = (b - a + 127) // 128
        assert torch.equal(t.exps[:, a // 128:a // 128 + n], other.exps[:, :n]), a


def test_an_inference_layer_of_more_rows_than_2_23():
    R, K, N = 2 ** 23 + 77, 16, 16
    print("linear", R, K, N, flush=True)
    x, w = randn(22, R, K).to(torch.bfloat16), ops().fp8_quantize(randn(23, N, K).to(torch.bfloat16), 128)
    y = ops().fp8_linear(x, w)
    for a in (0, 2 ** 22 - 64, 2 ** 23 - 100, R - 300):
        assert torch.equal(y[a:a + 300], ops().fp8_linear(x[a:a + 300], w)[:300]), a
