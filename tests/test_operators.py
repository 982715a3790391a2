"""Dense layer and layer norm (include/mace/operators.h, mace_inference.operators) against their
definitions in 64 bits.

Tolerances are bounds, derived from how a result is computed, not fitted:
  * u is half a step of the element type; the last rounding is at most u |result| (plus half the
    smallest subnormal).  f32: 2^-24, bf16: 2^-8, f16: 2^-11 (finfo.eps / 2).
  * A product accumulates in float.  With S = sum_k |p_k| |q_k|, every addition (the tensor
    pipe's may truncate) is off by at most 2^-23 of a partial sum <= S; there are fewer than
    K / 16 + 8 of them in sequence in 16-bit types (16 products enter at once), so the sum is
    within (K / 16 + 8) 2^-22 S.  f32 operands are split to 22 bits each (2 2^-22 S), the slab
    sums are added in float: within (K / 64 + 16) 2^-22 S.
  * Activations have slope at most 1.13 (gelu; silu 1.10) and are evaluated to 2^-20.
  * Gradients of 16-bit layers round dz to the type before the products: u |dz| more.
"""
import math
import random

import pytest

gpu = pytest.mark.gpu
TYPES = ["f32", "bf16", "f16"]
ACTS = [None, "silu", "gelu", "relu"]


@pytest.fixture(scope="module")
def op(library):
    from mace_inference import operators
    return operators


def dtype_of(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def half_step(dtype):
    import torch
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    import torch
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def normal(seed, *shape, dtype, scale=1.0, shift=0.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)


def act64(z, act):
    import torch
    f = torch.nn.functional
    return z if act is None else {"silu": f.silu, "gelu": f.gelu, "relu": f.relu}[act](z)


def slope64(z, act):
    import torch
    if act is None:
        return torch.ones_like(z)
    z = z.detach().clone().requires_grad_()
    return torch.autograd.grad(act64(z, act).sum(), z)[0]


def accumulation(dtype, K):
    import torch
    return (K / 64 + 16) * 2.0 ** -22 if dtype == torch.float32 else (K / 16 + 8) * 2.0 ** -22


def close(got, want, bound, what):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(err[bad][0]), float(bound.expand_as(err)[bad][0]))


def check_dense(op, x, w, bias, act, residual, keep):
    import torch
    got = op.dense(x, w, bias, act, residual, keep=keep)
    y, z = got if keep else (got, None)
    dt, u = x.dtype, half_step(x.dtype)
    K = x.shape[-1]
    z64 = x.double() @ w.double().t()
    S = x.double().abs() @ w.double().abs().t()
    if bias is not None:
        z64, S = z64 + bias.double(), S + bias.double().abs()
    a64 = act64(z64, act)
    y64 = a64 if residual is None else a64 + residual.double()
    dz = accumulation(dt, K) * S
    assert y.shape == y64.shape and y.dtype == dt and y.is_contiguous()
    # One more float rounding for the bias, the activation and the residual each: 2^-20 covers them.
    close(y, y64, 1.13 * dz + 2.0 ** -20 * (a64.abs() + y64.abs()) + u * (y64.abs() + 1.13 * dz) + tiny(dt), "y")
    if keep:
        close(z, z64, dz + u * (z64.abs() + dz) + tiny(dt), "z")
    return y, z


SHAPES = [  # rows, inputs, outputs
    (1, 1, 1), (1, 10, 64), (3, 64, 5), (17, 10, 64), (33, 64, 64), (5, 63, 65), (129, 65, 257), (200, 128, 130),
    (257, 130, 1), (1, 520, 300), (64, 1000, 72), (300, 256, 384), (1000, 72, 520), (130, 2056, 264), (2, 4096, 136),
]


@gpu
@pytest.mark.parametrize("act", ACTS, ids=str)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_dense(op, shape, dtype, act):
    M, K, N = shape
    dt = dtype_of(dtype)
    x, w = normal(1, M, K, dtype=dt), normal(2, N, K, dtype=dt, scale=K ** -0.5)
    b, r = normal(3, N, dtype=dt), normal(4, M, N, dtype=dt)
    check_dense(op, x, w, None, act, None, False)
    check_dense(op, x, w, b, act, r, True)


def check_dense_backward(op, dy, x, w, act, z, need=(True, True, True)):
    dx, dw, db = op.dense_backward(dy, x, w, act, z, need=need)
    import torch
    dt, u = x.dtype, half_step(x.dtype)
    M, N = dy.reshape(-1, dy.shape[-1]).shape
    K = x.shape[-1]
    flat = lambda t: t.reshape(-1, t.shape[-1]).double()  # noqa: E731
    g64 = flat(dy) if act is None else flat(dy) * slope64(flat(z), act)
    off = torch.zeros_like(g64) if act is None else 2.0 ** -20 * flat(dy).abs() * 1.2 + \
        (u * g64.abs() + tiny(dt) if dt != torch.float32 else 2.0 ** -23 * g64.abs())
    w64, x64 = w.double(), flat(x)
    if need[0]:
        want = (g64 @ w64).reshape(x.shape)
        S = ((g64.abs() + off) @ w64.abs()).reshape(x.shape)
        bound = (off @ w64.abs()).reshape(x.shape) + accumulation(dt, N) * S
        assert dx.shape == x.shape and dx.dtype == dt
        close(dx, want, bound + u * (want.abs() + bound) + tiny(dt), "dx")
    else:
        assert dx is None
    if need[1]:
        want, S = g64.t() @ x64, (g64.abs() + off).t() @ x64.abs()
        bound = off.t() @ x64.abs() + accumulation(dt, M) * S
        assert dw.shape == w.shape and dw.dtype == dt
        close(dw, want, bound + u * (want.abs() + bound) + tiny(dt), "dweight")
    else:
        assert dw is None
    if need[2]:
        want, S = g64.sum(0), g64.abs().sum(0)
        # Float sums over rows: fewer than M / 32 + 64 additions in sequence.
        bound = off.sum(0) + (M / 32 + 64) * 2.0 ** -24 * S
        close(db, want, bound + u * (want.abs() + bound) + tiny(dt), "dbias")
    else:
        assert db is None
    return dx, dw, db


@gpu
@pytest.mark.parametrize("act", ACTS, ids=str)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_dense_backward(op, shape, dtype, act):
    M, K, N = shape
    dt = dtype_of(dtype)
    x, w = normal(1, M, K, dtype=dt), normal(2, N, K, dtype=dt, scale=K ** -0.5)
    dy, z = normal(3, M, N, dtype=dt), normal(4, M, N, dtype=dt)
    check_dense_backward(op, dy, x, w, act, z)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_dense_backward_many_rows(op, dtype):
    """Few columns and many rows: the sum over rows is split over the device."""
    dt = dtype_of(dtype)
    x, w = normal(1, 20011, 24, dtype=dt), normal(2, 40, 24, dtype=dt)
    dy, z = normal(3, 20011, 40, dtype=dt), normal(4, 20011, 40, dtype=dt)
    for act in (None, "silu"):
        check_dense_backward(op, dy, x, w, act, z)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        check_dense_backward(op, dy, x, w, "silu", z, need)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(12, 9, 7), (3001, 63, 64), (20011, 24, 40), (3000, 200, 136)], ids=lambda s: "x".join(map(str, s)))
def test_dense_bias_gradient_sums_floats(op, shape, dtype):
    """dbias is a sum of floats, rounded once, whatever the layer's size: values of dz that the type rounds
    to nothing count, and none is rounded on its way (no u |dz| in the bound)."""
    M, K, N = shape
    dt = dtype_of(dtype)
    x, w = normal(1, M, K, dtype=dt), normal(2, N, K, dtype=dt)
    z = normal(4, M, N, dtype=dt)
    for dy in (normal(3, M, N, dtype=dt, scale=0.1, shift=1.0), normal(3, M, N, dtype=dt, scale=0.0, shift=2.0 ** -24)):
        for act, zs in (("silu", z), ("silu", z - 5), ("gelu", z)):
            _, _, db = op.dense_backward(dy, x, w, act, zs)
            d64 = dy.double()
            g64 = d64 * slope64(zs.double(), act)
            want, S = g64.sum(0), g64.abs().sum(0)
            # Slopes are off by at most 2^-20 of 1.13; fewer than M / 32 + 64 additions in sequence.
            bound = (1.13 * 2.0 ** -20 * d64.abs()).sum(0) + (M / 32 + 64) * 2.0 ** -24 * S
            close(db, want, bound + half_step(dt) * (want.abs() + bound) + tiny(dt) / 2, "dbias")


def spread(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


@gpu
@pytest.mark.parametrize("seed", range(30))
def test_dense_anywhere(op, seed):
    """Shapes drawn over the whole range, types, activations and options at random: few rows, few
    outputs, few inputs, several tiles per SM, sums cut into parts, rows that start anywhere."""
    rng = random.Random(seed)
    dt = dtype_of(rng.choice(TYPES))
    while True:
        M, K, N = spread(rng, 1, 6000), spread(rng, 1, 3000), spread(rng, 1, 3000)
        if rng.random() < 0.5:
            K, N = (K + 15) // 16 * 16, (N + 15) // 16 * 16
        if M * K * N < 4e9:
            break
    act = rng.choice(ACTS)
    x, w = normal(1, M, K, dtype=dt), normal(2, N, K, dtype=dt, scale=K ** -0.5)
    b = normal(3, N, dtype=dt) if rng.random() < 0.7 else None
    r = normal(4, M, N, dtype=dt) if rng.random() < 0.5 else None
    check_dense(op, x, w, b, act, r, rng.random() < 0.5)
    check_dense_backward(op, normal(5, M, N, dtype=dt), x, w, act, normal(6, M, N, dtype=dt))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 7, 8, 9])
def test_dense_few_rows_and_few_outputs(op, rows, dtype):
    dt = dtype_of(dtype)
    for K, N in ((33, 3), (256, 70), (1000, 1), (1001, 517), (5000, 64)):
        x, w, b = normal(1, rows, K, dtype=dt), normal(2, N, K, dtype=dt, scale=K ** -0.5), normal(3, N, dtype=dt)
        check_dense(op, x, w, b, "gelu", normal(4, rows, N, dtype=dt), True)
        x, w, b = normal(1, N, K, dtype=dt), normal(2, rows, K, dtype=dt, scale=K ** -0.5), normal(3, rows, dtype=dt)
        check_dense(op, x, w, b, "silu", normal(4, N, rows, dtype=dt), True)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(600, 203, 301), (300, 1003, 130), (130, 65, 1005), (400, 259, 63), (70, 4001, 9),
                                   (500, 63, 64), (500, 64, 63), (3000, 255, 15), (100003, 3, 5), (65, 1, 1), (64, 31, 1),
                                   (9, 400, 9), (1001, 11, 370), (18, 534, 94), (11, 3001, 96), (2, 9000, 230), (700, 90, 130)], ids=lambda s: "x".join(map(str, s)))
def test_dense_small_and_odd(op, shape, dtype):
    """Both sides of the limits under which operands of any alignment are read as they are, with
    rows further apart than they are long, and each gradient alone."""
    M, K, N = shape
    dt = dtype_of(dtype)
    x, w = normal(1, M, K + 3, dtype=dt)[:, 1:K + 1], normal(2, N, K + 2, dtype=dt, scale=K ** -0.5)[:, :K]
    b, r = normal(3, N, dtype=dt), normal(4, M, N + 5, dtype=dt)[:, 2:N + 2]
    z = normal(5, M, N + 1, dtype=dt)[:, :N]
    check_dense(op, x, w, b, "silu", r, True)
    check_dense(op, x, w, None, None, None, False)
    for need in ((True, True, True), (True, False, False), (False, True, False), (False, False, True)):
        check_dense_backward(op, r, x, w, "gelu", z, need)
    check_dense_backward(op, r, x, w, None, None)


@gpu
@pytest.mark.parametrize("shape", [(18943, 255, 16), (18944, 35, 9), (19001, 33, 16), (20001, 130, 17), (20001, 1001, 12),
                                   (40007, 13, 10), (40007, 12, 10), (30001, 31, 8), (90001, 41, 11), (19072, 98, 15)],
                         ids=lambda s: "x".join(map(str, s)))
def test_dense_many_odd_rows_and_few_outputs(op, shape):
    """Rows of floats that start anywhere, on both sides of the limits within which they are read as they
    are; infinities and NaN stay in their rows."""
    import torch
    M, K, N = shape
    f32 = dtype_of("f32")
    x, w = normal(1, M, K + 3, dtype=f32)[:, 1:K + 1], normal(2, N, K + 2, dtype=f32, scale=K ** -0.5)[:, :K]
    b, r = normal(3, N, dtype=f32), normal(4, M, N + 5, dtype=f32)[:, 2:N + 2]
    check_dense(op, x, w, b, "gelu", r, True)
    clean, _ = check_dense(op, x.contiguous(), w, None, None, None, False)
    assert torch.equal(op.dense(x, w), clean)
    bad = x.contiguous()
    bad[5, K - 1], bad[M - 1, 0], bad[70, 3] = math.inf, math.nan, -math.inf
    y = op.dense(bad, w)
    same = torch.ones(M, dtype=torch.bool, device="cuda")
    same[[5, 70, M - 1]] = False
    assert torch.equal(y[same], clean[same]) and y[M - 1].isnan().all()
    assert torch.equal(y[5].sign(), w[:, K - 1].sign()) and y[[5, 70]].isinf().all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_dense_larger(op, dtype):
    """Several tiles per SM with every part of the epilogue; a wide layer of few rows; a long sum."""
    dt = dtype_of(dtype)
    for M, K, N in ((5000, 200, 1200), (4097, 64, 2056), (40, 1024, 4104), (16, 20000, 24)):
        x, w = normal(1, M, K, dtype=dt), normal(2, N, K, dtype=dt, scale=K ** -0.5)
        b, r = normal(3, N, dtype=dt), normal(4, M, N, dtype=dt)
        for act, bias, residual, keep in ((None, None, None, False), ("gelu", b, None, True), ("silu", b, r, False),
                                          ("relu", None, r, True)):
            check_dense(op, x, w, bias, act, residual, keep)
        check_dense_backward(op, r, x, w, "gelu", normal(5, M, N, dtype=dt))
        check_dense_backward(op, r, x, w, None, None)


@gpu
def test_dense_offsets_beyond_32_bits(op):
    """Arrays whose elements lie more than 2^31 apart (rows of a wide buffer)."""
    import torch
    buf = torch.empty(5, 1 << 30, dtype=torch.bfloat16, device="cuda")
    x, r = buf[:, -136:-8], buf[:, 1 << 29:(1 << 29) + 64]
    x.copy_(normal(1, 5, 128, dtype=torch.bfloat16))
    r.copy_(normal(2, 5, 64, dtype=torch.bfloat16))
    w = normal(3, 64, 128, dtype=torch.bfloat16, scale=0.1)
    check_dense(op, x, w, None, "silu", r, False)
    mean, rstd = check_norm(op, x, None, None, 1e-5, None)
    check_norm_backward(op, normal(4, 5, 128, dtype=torch.bfloat16), x, mean, rstd, None, None, None)
    wide = torch.as_strided(buf.view(-1), (20, 128), (1 << 27, 1), 64)
    wide.copy_(normal(5, 20, 128, dtype=torch.bfloat16))
    check_dense(op, wide, w, None, None, None, True)
    check_dense_backward(op, normal(6, 20, 64, dtype=torch.bfloat16), wide, w, None, None)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_dense_strides_and_shapes(op, dtype):
    """Column blocks of one buffer, odd addresses and row distances, more than two dimensions,
    a transposed weight, an expanded gradient, a single vector."""
    import torch
    dt = dtype_of(dtype)
    buf = normal(5, 77, 403, dtype=dt)
    for first, K in ((0, 96), (1, 96), (3, 97), (8, 40)):
        x = buf[:, first:first + K]
        r = buf[:, 200 + first:200 + first + 72]
        w = normal(6, 73, 200, dtype=dt, scale=0.1)[1:, first:first + K]
        check_dense(op, x, w, None, "silu", r, True)
        dy, z = buf[:, 300 + first:372 + first], normal(7, 80, 500, dtype=dt)[2:79, first:first + 72]
        check_dense_backward(op, dy, x, w, "gelu", z)
    x3 = normal(8, 3, 5, 48, dtype=dt)
    w = normal(9, 48, 24, dtype=dt).t()
    check_dense(op, x3, w, None, None, None, False)
    check_dense(op, x3.transpose(0, 1), w, normal(10, 24, dtype=dt), "relu", None, True)
    check_dense_backward(op, torch.ones(24, dtype=dt, device="cuda").expand(3, 5, 24), x3, w, None, None)
    y = op.dense(x3[0, 0], w)
    assert y.shape == (24,) and torch.equal(y, op.dense(x3[0, :1], w)[0])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_dense_empty(op, dtype):
    import torch
    dt = dtype_of(dtype)
    w = normal(1, 6, 10, dtype=dt)
    x = torch.empty(0, 10, dtype=dt, device="cuda")
    y, z = op.dense(x, w, None, "silu", keep=True)
    assert y.shape == z.shape == (0, 6)
    dx, dw, db = op.dense_backward(y, x, w, "silu", z)
    assert dx.shape == (0, 10) and not dw.any() and not db.any() and dw.shape == (6, 10) and db.shape == (6,)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_dense_not_finite_values_stay_in_their_rows(op, dtype):
    """Rows (and weight rows) with infinities or NaN give what the sum in 64 bits gives, and all
    others what they give without them."""
    import torch
    dt = dtype_of(dtype)
    M, K, N = 150, 200, 140
    x, w = normal(1, M, K, dtype=dt), normal(2, N, K, dtype=dt)
    clean = op.dense(x, w)
    bad = x.clone()
    bad[3, 7], bad[40, 100], bad[41, 0], bad[149, 199] = math.inf, -math.inf, math.nan, math.inf
    bad[41, 1], bad[60, 10], bad[60, 150] = math.inf, math.inf, -math.inf
    wb = w.clone()
    wb[5, 3], wb[139, 199], wb[70, 70] = math.inf, math.nan, -math.inf
    wb[9, 7], wb[10, :] = 0.0, 0.0
    got = op.dense(bad, wb)
    # Finite values are replaced by their signs: the special ones decide the same.
    want = (bad.double()[:, None, :] * wb.double()[None]).sum(-1)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[want.isinf()].double(), want[want.isinf()])
    same = torch.ones(M, N, dtype=torch.bool, device="cuda")
    same[[3, 40, 41, 60, 149]] = False
    same[:, [5, 9, 10, 70, 139]] = False
    assert torch.equal(got[same], clean[same])
    # The same values in a gradient's operands.
    dy = normal(3, M, N, dtype=dt)
    dx, dw, _ = op.dense_backward(dy, bad, wb)
    want = (dy.double()[:, :, None] * wb.double()[None]).sum(1)
    assert torch.equal(dx.isnan(), want.isnan()) and torch.equal(dx[want.isinf()].double(), want[want.isinf()])
    want = (dy.double()[:, :, None] * bad.double()[:, None, :]).sum(0)
    assert torch.equal(dw.isnan(), want.isnan()) and torch.equal(dw[want.isinf()].double(), want[want.isinf()])


@gpu
def test_dense_f32_all_results_infinite(op):
    """Every result is an infinity, over long sums: each is summed again, which takes far longer
    than the products, and the waits inside the kernel outlast it."""
    import torch
    M, K, N = 9600, 32768, 128
    x = torch.ones(M, K, device="cuda")
    x[:, K - 1] = math.inf
    w = torch.ones(N, K, device="cuda")
    w[::2, K - 1] = -1.0
    want = torch.where(torch.arange(N, device="cuda") % 2 == 0, -math.inf, math.inf)
    assert torch.equal(op.dense(x, w), want.expand(M, N))


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", TYPES)
def test_activations_of_special_values(op, dtype, act):
    """Infinities, NaN and the type's largest values give what the formulas give, in every type."""
    import torch
    dt = dtype_of(dtype)
    big = torch.finfo(dt).max
    v = torch.tensor([math.inf, -math.inf, math.nan, big, -big, 0.0, 100.0, -100.0], dtype=dt, device="cuda")
    want, slope = act64(v.double(), act), slope64(v.double(), act)
    for k in (1, 64):  # both kinds of product; the first input carries the value
        x = torch.zeros(8, k, dtype=dt, device="cuda").repeat(20, 1)
        x[:, 0] = v.repeat(20)
        w = torch.zeros(16, k, dtype=dt, device="cuda")
        w[:, 0] = 1
        y, z = op.dense(x, w, None, act, keep=True)
        expected = want.to(dt).repeat(20)[:, None].expand(160, 16)
        assert torch.equal(y.isnan(), expected.isnan()) and torch.equal(z.isnan(), x[:, :1].isnan().expand(160, 16))
        # (1e-30: the floats' exponential overflows where the formula's value is far below that.)
        finite, bound = expected.isfinite(), (accumulation(dt, k) + 2 * half_step(dt)) * want.abs().repeat(20)[:, None] + 1e-30
        assert torch.equal(y[expected.isinf()], expected[expected.isinf()])
        close(y[finite], expected[finite].double(), bound.expand(160, 16)[finite], act)
        one = torch.ones(1, 16, dtype=dt, device="cuda")
        for i in range(8):
            _, _, db = op.dense_backward(one, x[i:i + 1], w, act, z[i:i + 1], need=(False, False, True))
            if slope[i].isnan():
                assert db.isnan().all()
            else:
                assert (db.double() - slope[i]).abs().max() <= 2 * half_step(dt)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_silu_far_below_zero(op, dtype):
    """SiLU and its slope relative to their own size, down to where they leave the type: z enters as the bias
    of a product of zeros."""
    import torch
    dt, u = dtype_of(dtype), half_step(dtype_of(dtype))
    z = torch.linspace(-104, 20, 2048, device="cuda").to(dt)
    x, w = torch.zeros(16, 8, dtype=dt, device="cuda"), torch.zeros(2048, 8, dtype=dt, device="cuda")
    y = op.dense(x, w, z, "silu")
    _, _, db = op.dense_backward(torch.ones(1, 2048, dtype=dt, device="cuda"), x[:1], w, "silu", z[None])
    z64 = z.double()
    # The exponential: 2 ulp in f32, |z| 2^-23 of its value in 16 bits; subnormal, it has steps of 2^-149.
    # Quotient and products: 6 ulp; the slope's 1 + z (1 - s) cancels near z = -1.28 only, to 2^-22.
    rel = 2.0 ** -20 + (z64.abs() * 2.0 ** -23 if dt != torch.float32 else 0)
    low = (z64.abs() + 1) * 2.0 ** -147 + tiny(dt)
    want = act64(z64, "silu")
    close(y, want.expand(16, 2048), (rel + u) * want.abs() + low, "silu")
    want = slope64(z64, "silu")
    close(db, want, (rel + u) * want.abs() + 2.0 ** -21 * ((z64 + 1.2785).abs() < 0.5) + low, "slope")


@gpu
def test_dense_f32_rows_of_any_magnitude(op):
    """Rows from 1e-25 to 1e25, and weights whose rows differ as much: the error stays relative to
    each row's own products."""
    import torch
    M, K, N = 300, 200, 130
    x = normal(1, M, K, dtype=torch.float32).double() * 10.0 ** torch.linspace(-25, 25, M, device="cuda").double()[:, None]
    w = normal(2, N, K, dtype=torch.float32).double() * 10.0 ** torch.linspace(-12, 12, N, device="cuda").double()[:, None]
    check_dense(op, x.float(), w.float(), None, None, None, False)
    check_dense_backward(op, normal(3, M, N, dtype=torch.float32), x.float(), w.float(), None, None,
                         need=(True, False, True))
    check_dense_backward(op, normal(3, M, N, dtype=torch.float32), x.float() * 1e-20, w.float(), None, None,
                         need=(False, True, True))


@gpu
@pytest.mark.parametrize("big", [1e3, 1e6, 1e8])
def test_dense_f32_values_beside_much_larger_ones(op, big):
    """A large value that meets a weight of zero: the others' products keep their bits, in the result and in
    both gradients (the bounds are relative to the products that are there)."""
    M, K, N = 300, 256, 200
    f32 = dtype_of("f32")
    x, w, dy = normal(1, M, K, dtype=f32), normal(2, N, K, dtype=f32), normal(3, M, N, dtype=f32)
    x[:, 70], w[:, 70] = big, 0.0
    check_dense(op, x, w, None, None, None, False)
    x, w = normal(1, M, K, dtype=f32), normal(2, N, K, dtype=f32)
    w[:, 30], x[:, 30] = big, 0.0
    check_dense(op, x, w, None, None, None, False)
    dy[:, 11], w[11], w[:, 30] = big, 0.0, 1.0
    check_dense_backward(op, dy, x, w, None, None, need=(True, False, False))
    dy[:, 11] = 1.0
    dy[40], x[40] = big, 0.0
    check_dense_backward(op, dy, x, w, None, None, need=(False, True, False))


@gpu
@pytest.mark.parametrize("shape", [(300, 64, 70), (300, 512, 200), (5000, 200, 40)], ids=lambda s: "x".join(map(str, s)))
def test_dense_f32_exact_sums_are_exact(op, shape):
    """Small integers: every partial sum is exact in floats, and so is the result.  A weight of ones on the
    diagonal returns x to the bits that the operands keep."""
    import torch
    M, K, N = shape
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w, dy = (torch.randint(-8, 9, s, device="cuda", generator=g).float() for s in ((M, K), (N, K), (M, N)))
    assert torch.equal(op.dense(x, w).double(), x.double() @ w.double().t())
    dx, dw, db = op.dense_backward(dy, x, w)
    assert torch.equal(dx.double(), dy.double() @ w.double()) and torch.equal(dw.double(), dy.double().t() @ x.double())
    assert torch.equal(db.double(), dy.double().sum(0))
    x = normal(2, M, K, dtype=torch.float32)
    y = op.dense(x, torch.eye(K, device="cuda"))
    assert ((y - x).abs() <= 2.0 ** -23 * x.abs()).all()


# ---------------------------------------------------------------- layer norm
def check_norm(op, x, gamma, beta, eps, act):
    import torch
    y, mean, rstd = op.layer_norm(x, gamma, beta, eps, act, keep=True)
    assert torch.equal(op.layer_norm(x, gamma, beta, eps, act).view(torch.uint8), y.view(torch.uint8))
    dt, u = x.dtype, half_step(x.dtype)
    x64 = x.double()
    m64 = x64.mean(-1)
    c64 = x64 - m64[..., None]
    var = c64.square().mean(-1)
    r64 = (var + eps) ** -0.5
    std = var.sqrt()
    # The centred values carry their own rounding (2^-24) and the correction's; the row sums at most
    # n / 1024 + 48 additions in sequence.
    rel = (x.shape[-1] / 1024 + 64) * 2.0 ** -24
    close(mean, m64, 2.0 ** -23 * m64.abs() + rel * std + 1e-37, "mean")
    close(rstd, r64, 2 * rel * r64, "rstd")
    g64 = torch.ones_like(x64[..., :]) if gamma is None else gamma.double()
    b64 = torch.zeros_like(x64) if beta is None else beta.double()
    xh = c64 * r64[..., None]
    z64 = xh * g64 + b64
    y64 = act64(z64, act)
    dz = (3 * rel * (xh.abs() + 1) * g64.abs() + 2.0 ** -23 * b64.abs())
    assert y.dtype == dt and y.shape == x.shape
    close(y, y64, 1.13 * dz + 2.0 ** -20 * y64.abs() + u * (y64.abs() + 1.13 * dz) + tiny(dt), "y")
    return mean, rstd


def check_norm_backward(op, dy, x, mean, rstd, gamma, beta, act, need=(True, True, True)):
    import torch
    dx, dg, db = op.layer_norm_backward(dy, x, mean, rstd, gamma, beta, act, need=need)
    dt, u = x.dtype, half_step(x.dtype)
    n = x.shape[-1]
    two = lambda t: t.reshape(-1, n).double()  # noqa: E731
    r = rstd.reshape(-1, 1).double()
    xh = (two(x) - mean.reshape(-1, 1).double()) * r
    g64 = torch.ones(n, device="cuda").double() if gamma is None else gamma.double()
    b64 = torch.zeros(n, device="cuda").double() if beta is None else beta.double()
    z = xh * g64 + b64
    zoff = 2.0 ** -22 * (xh * g64).abs() + 2.0 ** -23 * z.abs()
    d = two(dy)
    dz = d * slope64(z, act)
    # slopes of slopes are below 1.6 / 2; relu steps where z may round to either side of zero.
    off = torch.zeros_like(d) if act is None else d.abs() * (2.0 ** -20 * 1.2 + 0.8 * zoff)
    if act == "relu":
        off = off + d.abs() * (z.abs() <= zoff)
    g, goff = dz * g64, off * g64.abs() + 2.0 ** -24 * (dz * g64).abs()
    rel = (n / 1024 + 64) * 2.0 ** -24
    if need[0]:
        mg, mgx = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
        mgo = goff.mean(1, keepdim=True) + rel * g.abs().mean(1, keepdim=True)
        mgxo = (goff * xh.abs()).mean(1, keepdim=True) + 2 * rel * (g * xh).abs().mean(1, keepdim=True)
        want = r * (g - mg - xh * mgx)
        bound = r * (goff + mgo + xh.abs() * mgxo + 2.0 ** -21 * (g.abs() + mg.abs() + (xh * mgx).abs()))
        close(dx.reshape(-1, n), want, bound + u * (want.abs() + bound) + tiny(dt), "dx")
    rows = d.shape[0]
    seq = (rows / 64 + 128) * 2.0 ** -24
    if need[1]:
        want, S = (dz * xh).sum(0), (dz * xh).abs().sum(0)
        bound = (off * xh.abs()).sum(0) + (seq + 2.0 ** -22) * S
        close(dg, want, bound + u * (want.abs() + bound) + tiny(dt), "dgamma")
    if need[2]:
        want, S = dz.sum(0), dz.abs().sum(0)
        bound = off.sum(0) + (seq + 2.0 ** -24) * S
        close(db, want, bound + u * (want.abs() + bound) + tiny(dt), "dbeta")


NORM_SHAPES = [(1, 1), (3, 2), (5, 7), (1000, 64), (17, 64), (2, 65), (33, 128), (9, 250), (40, 511), (7, 1000),
               (300, 1024), (5, 1032), (12, 2053), (3, 4096), (11, 5120), (2, 8192), (3, 10001), (2, 16384), (3, 20000),
               (2, 33001), (2, 40000)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_layer_norm(op, shape, dtype):
    dt = dtype_of(dtype)
    M, n = shape
    x = normal(1, M, n, dtype=dt, scale=1.7, shift=0.4)
    gamma, beta = normal(2, n, dtype=dt, scale=0.3, shift=1.0), normal(3, n, dtype=dt, scale=0.3)
    dy = normal(4, M, n, dtype=dt)
    for act in ACTS:
        mean, rstd = check_norm(op, x, gamma, beta, 1e-5, act)
        check_norm_backward(op, dy, x, mean, rstd, gamma, beta, act)
    check_norm(op, x, None, None, 1e-5, None)
    check_norm_backward(op, dy, x, mean, rstd, None, None, None)
    check_norm(op, x, gamma, None, 1e-3, "silu")
    check_norm_backward(op, dy, x, mean, rstd, gamma, None, "silu")
    check_norm_backward(op, dy, x, mean, rstd, None, beta, "gelu")


@gpu
@pytest.mark.parametrize("seed", range(30))
def test_layer_norm_anywhere(op, seed):
    """Shapes drawn over the whole range, with types, activations and parameters at random; half of the
    arrays are column blocks of wider ones."""
    rng = random.Random(seed)
    dt = dtype_of(rng.choice(TYPES))
    M, n = spread(rng, 1, 5000), spread(rng, 8, 14000)
    M = min(M, 4000000 // n)
    if rng.random() < 0.4:
        n = (n + 7) // 8 * 8
    wide = n + rng.choice([0, 0, 8, 3])
    x = normal(1, M, wide, dtype=dt, scale=1.7, shift=0.4)[:, :n]
    dy = normal(4, M, wide, dtype=dt)[:, wide - n:]
    gamma = normal(2, n, dtype=dt, scale=0.3, shift=1.0) if rng.random() < 0.8 else None
    beta = normal(3, n, dtype=dt, scale=0.3) if rng.random() < 0.8 else None
    act = rng.choice(ACTS)
    mean, rstd = check_norm(op, x, gamma, beta, 1e-5, act)
    check_norm_backward(op, dy, x, mean, rstd, gamma, beta, act)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_many_rows_and_strides(op, dtype):
    dt = dtype_of(dtype)
    x, dy = normal(1, 30011, 64, dtype=dt), normal(2, 30011, 64, dtype=dt)
    gamma, beta = normal(3, 64, dtype=dt), normal(4, 64, dtype=dt)
    mean, rstd = check_norm(op, x, gamma, beta, 1e-5, "silu")
    check_norm_backward(op, dy, x, mean, rstd, gamma, beta, "silu")
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        check_norm_backward(op, dy, x, mean, rstd, gamma, beta, "silu", need)
    buf = normal(5, 90, 500, dtype=dt)
    for first, n in ((0, 96), (1, 96), (8, 97), (16, 200)):
        xs, ds = buf[:, first:first + n], buf[:, 250 + first:250 + first + n]
        g, b = normal(6, 300, dtype=dt)[first:first + n], normal(7, 300, dtype=dt)[:2 * n:2][:n]
        g, b = g[:n], b[:n] if b.numel() >= n else g
        mean, rstd = check_norm(op, xs, g, b, 1e-5, "gelu")
        check_norm_backward(op, ds, xs, mean, rstd, g, b, "gelu")
    x3 = normal(8, 4, 6, 40, dtype=dt).transpose(0, 1)
    mean, rstd = check_norm(op, x3, None, None, 1e-5, None)
    check_norm_backward(op, normal(9, 6, 4, 40, dtype=dt), x3, mean, rstd, None, None, None)
    check_norm(op, x3[0, 0], None, None, 1e-5, None)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(40001, 131, 131), (3001, 333, 333), (701, 2053, 2053), (1201, 333, 340),
                                   (5, 16395, 16395), (3, 40000, 40000), (301, 1024, 1024)],
                         ids=lambda s: "x".join(map(str, s)))
def test_layer_norm_gradients_left_out(op, shape, dtype):
    """Each way to leave gradients out, on rows that form spans (several rows, several spans a block; a row
    a span), on rows too wide for registers and on aligned ones: what is asked for does not change."""
    import torch
    dt = dtype_of(dtype)
    M, n, ld = shape
    x, dy = normal(1, M, ld, dtype=dt)[:, :n], normal(2, M, ld, dtype=dt)[:, :n]
    gamma, beta = normal(3, n, dtype=dt), normal(4, n, dtype=dt)
    mean, rstd = check_norm(op, x, gamma, beta, 1e-5, "silu")
    check_norm_backward(op, dy, x, mean, rstd, gamma, beta, "silu")
    full = op.layer_norm_backward(dy, x, mean, rstd, gamma, beta, "silu")
    for need in ((False, True, True), (False, True, False), (False, False, True), (True, False, False), (True, True, False)):
        got = op.layer_norm_backward(dy, x, mean, rstd, gamma, beta, "silu", need)
        for wanted, a, b in zip(need, got, full):
            assert torch.equal(a, b) if wanted else a is None


@gpu
def test_layer_norm_far_from_zero(op):
    """Rows of mean 1e4 and standard deviation 1: the variance is taken about the row's own mean."""
    import torch
    x = normal(1, 50, 1000, dtype=torch.float32, shift=1e4)
    check_norm(op, x, None, None, 1e-5, None)
    x = normal(2, 50, 4096, dtype=torch.float32, scale=1e-3, shift=-100.0)
    check_norm(op, x, None, None, 1e-12, None)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [8, 56, 127, 504, 896, 1000, 3584, 7160, 16392])
def test_layer_norm_rows_with_little_spread(op, n, dtype):
    """Constant rows far from zero, and rows of which one element is a step away: where rows start, and
    with them the kernel, makes no difference."""
    import torch
    dt = dtype_of(dtype)
    values = [0.1, -1536.0, 7168.0, 30000.0, 49152.0] + [2031616.0] * (dt != torch.float16)
    x = torch.tensor(values + values, device="cuda").to(dt)[:, None].repeat(1, n)
    for k in range(len(values)):
        x[k, n // 3] = torch.nextafter(x[k, 0], torch.tensor(math.inf, dtype=dt, device="cuda"))
    gamma, beta = normal(1, n, dtype=dt, scale=0.2, shift=1.0), normal(2, n, dtype=dt)
    anywhere = torch.empty(x.shape[0], n + 1, dtype=dt, device="cuda")[:, 1:]
    for rows in (x, anywhere.copy_(x)):
        mean, rstd = check_norm(op, rows, None, None, 1e-5, None)
        assert torch.equal(mean[len(values):], x[len(values):, 0].float())
        check_norm(op, rows, gamma, beta, 1e-5, "silu")


@gpu
@pytest.mark.parametrize("n", [56, 1000, 4096, 16384, 32768])
@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_rows_that_begin_far_from_the_rest(op, n, dtype):
    """One value decides a row's mean and spread, in the first place, behind it, and in the last."""
    dt = dtype_of(dtype)
    x = normal(1, 12, n, dtype=dt)
    for k, at in enumerate((0, 1, n // 2, n - 1)):
        x[3 * k, at], x[3 * k + 1, at], x[3 * k + 2, at] = 60000.0, -300.0, 20.0
    mean, rstd = check_norm(op, x, None, None, 1e-5, None)
    check_norm_backward(op, normal(2, 12, n, dtype=dt), x, mean, rstd, None, None, None)


@gpu
@pytest.mark.parametrize("n", [64, 2053, 40000])
@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_special_rows(op, dtype, n):
    import torch
    dt = dtype_of(dtype)
    x = normal(1, 9, n, dtype=dt)
    clean = op.layer_norm(x)
    x[1, 5], x[3, 0], x[6, n - 1] = math.inf, math.nan, -math.inf
    x[8] = 0.75  # constant: the variance is 0
    y, mean, rstd = op.layer_norm(x, keep=True)
    assert y[[1, 3, 6]].isnan().all() and not y[8].any()
    assert torch.equal(y[[0, 2, 4, 5, 7]], clean[[0, 2, 4, 5, 7]])
    assert mean[8] == 0.75 and abs(rstd[8].item() - 1e-5 ** -0.5) < 1e-4
    dx, dg, db = op.layer_norm_backward(normal(2, 9, n, dtype=dt), x, mean, rstd)
    assert dx[[1, 3, 6]].isnan().all() and dx[[0, 2, 4, 5, 7, 8]].isfinite().all()
    assert dg.isnan().all() and db.isfinite().all()


@gpu
@pytest.mark.parametrize("n", [8192, 8196, 12287, 12288, 12289, 16384, 16385, 16392])
@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_many_wide_rows(op, dtype, n):
    """Both sides of the lengths at which rows stop being held, with more rows than partial sums."""
    dt = dtype_of(dtype)
    x, dy, gamma = normal(1, 200, n, dtype=dt), normal(2, 200, n, dtype=dt), normal(3, n, dtype=dt)
    mean, rstd = check_norm(op, x, gamma, None, 1e-5, None)
    check_norm_backward(op, dy, x, mean, rstd, gamma, None, None)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_empty(op, dtype):
    import torch
    dt = dtype_of(dtype)
    x = torch.empty(0, 24, dtype=dt, device="cuda")
    y, mean, rstd = op.layer_norm(x, keep=True)
    dx, dg, db = op.layer_norm_backward(y, x, mean, rstd)
    assert y.shape == dx.shape == (0, 24) and mean.shape == (0,) and not dg.any() and not db.any()


# ---------------------------------------------------------------- together, streams, graphs
def radial_forward(op, x, layers, act="silu"):
    """Linear, LayerNorm + SiLU per hidden layer, Linear: the output and what the backward needs."""
    kept = []
    for w, b, gamma, beta in layers[:-1]:
        h = op.dense(x, w, b)
        y, mean, rstd = op.layer_norm(h, gamma, beta, activation=act, keep=True)
        kept.append((x, h, mean, rstd))
        x = y
    w, b = layers[-1]
    kept.append(x)
    return op.dense(x, w, b), kept


def radial_backward(op, dy, layers, kept, act="silu"):
    w, _ = layers[-1]
    dx, dw, db = op.dense_backward(dy, kept[-1], w)
    grads = [(dw, db)]
    for (w, b, gamma, beta), (x, h, mean, rstd) in zip(layers[-2::-1], kept[-2::-1]):
        dh, dgamma, dbeta = op.layer_norm_backward(dx, h, mean, rstd, gamma, beta, act)
        dx, dw, db = op.dense_backward(dh, x, w)
        grads.append((dw, db, dgamma, dbeta))
    return dx, grads[::-1]


def make_network(dtype, widths=(10, 64, 64, 64, 1280), seed=20):
    layers = []
    for k, (i, o) in enumerate(zip(widths[:-1], widths[1:])):
        layer = (normal(seed + 4 * k, o, i, dtype=dtype, scale=i ** -0.5), normal(seed + 4 * k + 1, o, dtype=dtype, scale=0.1))
        if k + 2 < len(widths):
            layer += (normal(seed + 4 * k + 2, o, dtype=dtype, scale=0.1, shift=1.0), normal(seed + 4 * k + 3, o, dtype=dtype, scale=0.1))
        layers.append(layer)
    return layers


def reference_network(x, layers):
    """The network in 64 bits with autograd: (output, leaves)."""
    import torch
    leaves = [x.double().requires_grad_()] + [v.double().requires_grad_() for layer in layers for v in layer]
    it = iter(leaves[1:])
    h = leaves[0]
    for layer in layers[:-1]:
        w, b, gamma, beta = (next(it) for _ in layer)
        h = torch.nn.functional.silu(torch.nn.functional.layer_norm(h @ w.t() + b, (w.shape[0],), gamma, beta))
    w, b = (next(it) for _ in layers[-1])
    return h @ w.t() + b, leaves


@gpu
@pytest.mark.parametrize("dtype,tol", [("f32", 2e-5), ("bf16", 0.05), ("f16", 6e-3)])
def test_radial_network(op, dtype, tol):
    """The MH1 radial network (10-64-64-64-1280) over 1000 edges, its output and all gradients,
    against the same network in 64 bits.  A layer adds a few roundings of relative size u to its
    values (f32: 2^-20 from the products); through three layers, forward and back, with
    condition numbers of a few, 2-norm errors stay below about 12 u (f32: 2e-5 ~ 20 2^-20)."""
    import torch
    dt = dtype_of(dtype)
    layers = make_network(dt)
    x, dy = normal(1, 1000, 10, dtype=dt), normal(2, 1000, 1280, dtype=dt)
    y, kept = radial_forward(op, x, layers)
    dx, grads = radial_backward(op, dy, layers, kept)
    y64, leaves = reference_network(x, layers)
    want = torch.autograd.grad(y64, leaves, dy.double())
    got = [dx] + [g for layer in grads for g in layer]
    for a, b in zip([y] + got, [y64.detach()] + list(want)):
        assert a.shape == b.shape
        err = ((a.double() - b).norm() / b.norm()).item()
        assert err < tol, err


@gpu
def test_radial_network_against_differences(op):
    """The loss sum(y dy) moved along each leaf's direction: central differences in 64 bits of the
    same network agree with the gradients' inner products."""
    import torch
    layers = make_network(torch.float32, widths=(10, 64, 64, 96))
    x, dy = normal(1, 200, 10, dtype=torch.float32), normal(2, 200, 96, dtype=torch.float32)
    _, kept = radial_forward(op, x, layers)
    dx, grads = radial_backward(op, dy, layers, kept)
    got = [dx] + [g for layer in grads for g in layer]
    flat = [x] + [v for layer in layers for v in layer]
    for k, (leaf, grad) in enumerate(zip(flat, got)):
        d = normal(50 + k, *leaf.shape, dtype=torch.float32).double()
        loss = []
        for h in (1e-4, -1e-4):
            moved = [v.double() + h * d if i == k else v.double() for i, v in enumerate(flat)]
            it = iter(moved[1:])
            y, _ = reference_network(moved[0], [tuple(next(it) for _ in layer) for layer in layers])
            loss.append((y.detach() * dy.double()).sum().item())
        slope, inner = (loss[0] - loss[1]) / 2e-4, (grad.double() * d).sum().item()
        scale = grad.double().norm().item() * d.norm().item()
        # f32 gradients to 2e-5 of their norm; the difference's own error is h^2 times the third
        # derivative (a few times the loss's scale here): 1e-6 of it at most.
        assert abs(slope - inner) <= 3e-5 * scale, (k, slope, inner)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_repeated_calls_give_equal_bits(op, dtype):
    import torch
    dt = dtype_of(dtype)
    layers = make_network(dt, widths=(10, 64, 200))
    x, dy = normal(1, 5003, 10, dtype=dt), normal(2, 5003, 200, dtype=dt)

    def once():
        y, kept = radial_forward(op, x, layers)
        dx, grads = radial_backward(op, dy, layers, kept)
        return [y, dx] + [g for layer in grads for g in layer]
    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


@gpu
def test_streams(op):
    """Calls on two streams at once, on tensors made on another stream."""
    import torch
    layers = make_network(torch.float32, widths=(10, 64, 64, 1280))
    xs = [normal(k, 3000, 10, dtype=torch.float32) for k in range(2)]
    dys = [normal(9 + k, 3000, 1280, dtype=torch.float32) for k in range(2)]

    def once(k):
        y, kept = radial_forward(op, xs[k], layers)
        dx, grads = radial_backward(op, dys[k], layers, kept)
        return [y, dx] + [g for layer in grads for g in layer]
    want = [once(k) for k in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(3):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k] = once(k)
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for a, b in zip(want[k], got[k]))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_captured_graphs(op, dtype):
    """A forward and backward pass captured, replayed on new inputs, and two such graphs replayed in
    turn: the results equal the eager calls'."""
    import torch
    dt = dtype_of(dtype)
    layers = make_network(dt, widths=(10, 64, 64, 200))
    static = [[normal(k, 700, 10, dtype=dt), normal(9 + k, 700, 200, dtype=dt)] for k in range(2)]

    def once(x, dy):
        y, kept = radial_forward(op, x, layers)
        dx, grads = radial_backward(op, dy, layers, kept)
        return [y, dx] + [g for layer in grads for g in layer]
    once(*static[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(once(*static[k]))
        graphs.append(g)
    for turn in range(2):
        for k in range(2):
            static[k][0].copy_(normal(30 + 2 * turn + k, 700, 10, dtype=dt))
            static[k][1].copy_(normal(40 + 2 * turn + k, 700, 200, dtype=dt))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], once(*static[k])))


@gpu
def test_in_place_and_untouched_memory(op, library):
    """Through the C entries: y over its residual, layer norm over its input, dx over dy; memory
    between the rows of a strided output, and behind the last row, stays as it was."""
    import torch
    lib = op._library()[0]
    s = torch.cuda.current_stream().cuda_stream
    for dt, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        M, K, N, ld = 70, 48, 40, 56
        x, w, r = normal(1, M, K, dtype=dt), normal(2, N, K, dtype=dt), normal(3, M, N, dtype=dt)
        want = op.dense(x, w, None, "silu", r)
        buf = torch.full((M + 2, ld), 7.0, dtype=dt, device="cuda")
        buf[:M, :N] = r
        size = lib.mace_dense_workspace(code, M, K, N, x.data_ptr(), K, w.data_ptr(), K)
        ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        assert lib.mace_dense(code, M, K, N, x.data_ptr(), K, w.data_ptr(), K, None, 1, buf.data_ptr(), ld,
                              buf.data_ptr(), ld, None, 0, ws.data_ptr(), size, s) == 0
        assert torch.equal(buf[:M, :N], want) and (buf[:, N:] == 7).all() and (buf[M:] == 7).all()
        want, mean, rstd = op.layer_norm(r, keep=True)
        buf[:M, :N] = r
        assert lib.mace_layer_norm(code, M, N, buf.data_ptr(), ld, None, None, 1e-5, 0, buf.data_ptr(), ld, None, None,
                                   s) == 0
        assert torch.equal(buf[:M, :N], want) and (buf[:, N:] == 7).all() and (buf[M:] == 7).all()
        dy = normal(4, M, N, dtype=dt)
        want, dg, db = op.layer_norm_backward(dy, r, mean, rstd)
        buf[:M, :N] = dy
        size = lib.mace_layer_norm_backward_workspace(code, M, N)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        g2, b2 = torch.empty_like(dg), torch.empty_like(db)
        assert lib.mace_layer_norm_backward(code, M, N, buf.data_ptr(), ld, r.data_ptr(), N, mean.data_ptr(),
                                            rstd.data_ptr(), None, None, 0, buf.data_ptr(), ld, g2.data_ptr(),
                                            b2.data_ptr(), ws.data_ptr(), size, s) == 0
        assert torch.equal(buf[:M, :N], want) and (buf[:, N:] == 7).all() and (buf[M:] == 7).all()
        assert torch.equal(g2, dg) and torch.equal(b2, db)


# ---------------------------------------------------------------- refusals (no GPU needed)
def call_dense(lib, type=0, rows=4, inputs=8, outputs=16, x=0x10000, ldx=8, w=0x20000, ldw=8, bias=None, act=0,
               r=None, ldr=0, y=0x30000, ldy=16, z=None, ldz=0, ws=None, size=0):
    code = lib.mace_dense(type, rows, inputs, outputs, x, ldx, w, ldw, bias, act, r, ldr, y, ldy, z, ldz, ws, size, None)
    return code, lib.mace_last_error().decode()


def call_dense_backward(lib, type=0, rows=100, inputs=8, outputs=16, dy=0x10000, lddy=16, x=0x20000, ldx=8, w=0x30000,
                        ldw=8, act=0, z=None, ldz=0, dx=0x40000, lddx=8, dw=0x50000, lddw=8, db=0x60000, ws=0x1000000,
                        size=1 << 24):
    code = lib.mace_dense_backward(type, rows, inputs, outputs, dy, lddy, x, ldx, w, ldw, act, z, ldz, dx, lddx, dw,
                                   lddw, db, ws, size, None)
    return code, lib.mace_last_error().decode()


def call_norm(lib, type=0, rows=4, width=16, x=0x10000, ldx=16, g=None, b=None, eps=1e-5, act=0, y=0x20000, ldy=16,
              mean=None, rstd=None):
    code = lib.mace_layer_norm(type, rows, width, x, ldx, g, b, eps, act, y, ldy, mean, rstd, None)
    return code, lib.mace_last_error().decode()


def call_norm_backward(lib, type=0, rows=4, width=16, dy=0x10000, lddy=16, x=0x20000, ldx=16, mean=0x30000,
                       rstd=0x30100, g=None, b=None, act=0, dx=0x40000, lddx=16, dg=0x50000, db=0x60000, ws=0x1000000,
                       size=1 << 24):
    code = lib.mace_layer_norm_backward(type, rows, width, dy, lddy, x, ldx, mean, rstd, g, b, act, dx, lddx, dg, db,
                                        ws, size, None)
    return code, lib.mace_last_error().decode()


REFUSED = [
    (call_dense, dict(type=3), "Invalid element type"),
    (call_dense, dict(type=-1), "Invalid element type"),
    (call_dense, dict(act=4), "Invalid activation"),
    (call_dense, dict(rows=-1), "Invalid row count"),
    (call_dense, dict(rows=1 << 31), "Invalid row count"),
    (call_dense, dict(inputs=0), "Invalid row length"),
    (call_dense, dict(outputs=(1 << 28) + 1), "Invalid row length"),
    (call_dense, dict(x=None), "Null array: x"),
    (call_dense, dict(w=None), "Null array: weight"),
    (call_dense, dict(y=None), "Null array: y"),
    (call_dense, dict(x=0x10002), "Misaligned array: x"),
    (call_dense, dict(ldx=7), "Invalid row distance: x"),
    (call_dense, dict(ldy=15), "Invalid row distance: y"),
    (call_dense, dict(r=0x40000, ldr=15), "Invalid row distance: residual"),
    (call_dense, dict(ldx=1 << 33), "Invalid row distance: x"),
    (call_dense, dict(rows=(1 << 31) - 1, ldx=1 << 32), "Array too large: x"),
    (call_dense, dict(y=0x10010), "overlaps"),
    (call_dense, dict(z=0x30040, ldz=16), "overlaps"),
    (call_dense, dict(r=0x30000, ldr=17), "overlaps"),
    (call_dense, dict(bias=0x30004), "overlaps"),
    (call_dense_backward, dict(act=1), "Null array: z"),
    (call_dense_backward, dict(dy=None), "Null array: dy"),
    (call_dense_backward, dict(size=0), "Workspace too small"),
    (call_dense_backward, dict(ws=None), "Workspace too small"),
    (call_dense_backward, dict(ws=0x1000008), "Misaligned workspace"),
    (call_dense_backward, dict(dx=0x10000), "overlaps"),
    (call_dense_backward, dict(dx=0x1000000), "overlaps"),
    (call_dense_backward, dict(db=0x50020), "overlaps"),
    (call_dense_backward, dict(dw=0x30000), "overlaps"),
    (call_norm, dict(eps=-1.0), "Invalid eps"),
    (call_norm, dict(eps=math.nan), "Invalid eps"),
    (call_norm, dict(mean=0x50000), "mean and rstd go together"),
    (call_norm, dict(width=0), "Invalid row length"),
    (call_norm, dict(y=0x10040), "overlaps"),
    (call_norm, dict(y=0x10000, ldy=17), "overlaps"),
    (call_norm, dict(x=None), "Null array: x"),
    (call_norm_backward, dict(mean=None), "Null array: mean"),
    (call_norm_backward, dict(size=0), "Workspace too small"),
    (call_norm_backward, dict(dx=0x20000), "overlaps"),
    (call_norm_backward, dict(dg=0x60000), "overlaps"),
    (call_norm_backward, dict(type=7), "Invalid element type"),
]


@pytest.mark.parametrize("call,wrong,message", REFUSED, ids=lambda v: v.__name__ if callable(v) else str(v)[:40])
def test_refusals(op, call, wrong, message):
    """Wrong arguments are refused before anything is launched (the addresses are not real)."""
    lib = op._library()[0]
    code, error = call(lib, **wrong)
    assert code == -1 and message in error, error


@pytest.mark.parametrize("type,held", [(0, 12288), (1, 16384), (2, 16384)])
def test_workspace_of_wide_rows(op, type, held):
    """Rows longer than any kernel holds at once have at most 32 partial sums of the parameters' gradients."""
    size = op._library()[0].mace_layer_norm_backward_workspace
    assert size(type, 2000, held) == 1184 * 2 * held * 4
    assert size(type, 2000, held + 1) == 32 * 2 * (held + 1) * 4
    assert size(type, 3, 1 << 20) == 3 * 2 * (1 << 20) * 4


def test_no_rows_is_no_work(op):
    lib = op._library()[0]
    assert call_dense(lib, rows=0, x=None, y=None)[0] == 0
    assert call_norm(lib, rows=0, x=None, y=None)[0] == 0
    assert call_dense_backward(lib, rows=0, dy=None, dw=None, db=None, dx=None, size=0, ws=None)[0] == 0
    assert lib.mace_dense_workspace(0, 0, 8, 8, None, 8, None, 8) == 0


def test_python_refusals(op):
    import torch
    x, w = torch.ones(3, 8), torch.ones(5, 8)
    with pytest.raises(ValueError, match="CUDA"):
        op.dense(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        op.layer_norm(x)
    with pytest.raises(TypeError, match="float32"):
        op.dense(x.double(), w)
    with pytest.raises(TypeError, match="torch tensor"):
        op.layer_norm([1.0])
    with pytest.raises(ValueError, match="activation"):
        op.dense(x, w, activation="tanh")
    with pytest.raises(ValueError, match="activation"):
        op.layer_norm(x, activation=["silu"])


@gpu
def test_python_refusals_on_the_gpu(op):
    import torch
    x, w, b = torch.ones(3, 8, device="cuda"), torch.ones(5, 8, device="cuda"), torch.ones(5, device="cuda")
    y = torch.ones(3, 5, device="cuda")
    for wrong in (lambda: op.dense(x, w.t()), lambda: op.dense(x, b), lambda: op.dense(x, w, x[0]),
                  lambda: op.dense(x, w.cpu()), lambda: op.dense(x, w, residual=x), lambda: op.dense(x[0, 0], w),
                  lambda: op.dense_backward(x, x, w), lambda: op.dense_backward(y, x, w, "silu"),
                  lambda: op.layer_norm(x, b), lambda: op.layer_norm_backward(x, x, b, b)):
        with pytest.raises(ValueError):
            wrong()
    for wrong in (lambda: op.dense(x, w.half()), lambda: op.dense(x, w, b.bfloat16()),
                  lambda: op.layer_norm_backward(x, x, x[:, 0].half(), x[:, 0])):
        with pytest.raises(TypeError):
            wrong()
    with pytest.raises(RuntimeError, match="row length"):
        op.dense(x[:, :0], w[:, :0])
    with pytest.raises(RuntimeError, match="eps"):
        op.layer_norm(x, eps=-1.0)
    torch.cuda.synchronize()


@gpu
def test_results_without_history_are_announced(op):
    """A forward call on tensors that require gradients, with autograd on, warns; the values are the same, and
    without autograd, or on detached tensors, and in the backward calls, nothing is said."""
    import warnings

    import torch
    x, w = normal(1, 20, 16, dtype=torch.float32), normal(2, 24, 16, dtype=torch.float32)
    p, g = torch.nn.Parameter(w), torch.nn.Parameter(x[0].clone())
    for call, plain in ((lambda: op.dense(x, p), lambda: op.dense(x, w)),
                        (lambda: op.dense(x.clone().requires_grad_(), w), lambda: op.dense(x, w)),
                        (lambda: op.layer_norm(x, g), lambda: op.layer_norm(x, g.detach()))):
        with pytest.warns(UserWarning, match="no autograd graph"):
            y = call()
        assert not y.requires_grad
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            assert torch.equal(y, plain())
            with torch.no_grad():
                assert torch.equal(y, call())
            op.dense_backward(normal(3, 20, 24, dtype=torch.float32), x, p)


# ---------------------------------------------------------------- schedules (no GPU needed)
@pytest.mark.parametrize("width", [64, 128])
def test_float_product_scales_are_read_before_they_are_written_again(width):
    """The float product's schedule as a graph of what waits for what: the split of slab n writes the
    scale slot of slab n - slots, so every drain warp's reads of that slab come before it."""
    import pathlib
    import re
    source = (pathlib.Path(__file__).parent.parent / "lasp-pis_b200/csrc/mace/dense_gemm32.cu").read_text()
    number = {}
    for name in ("stages", "buffers", "slots"):
        body = re.search(rf"constexpr int {name}\(\) {{ return (.*?); }}", source).group(1)
        body = re.sub(r"BN == 64 \? (\d+) : (\d+)", lambda m: m.group(1 if width == 64 else 2), body)
        number[name] = eval(re.sub(r"(\w+)<BN>\(\)", lambda m: str(number[m.group(1)]), body))
    stages, buffers, slots = number["stages"], number["buffers"], number["slots"]
    warps, slabs = 8, 40
    after = {}  # event -> events it comes after
    for n in range(slabs):
        # Loads of slab n are started by one drain warp, in turn, that has seen the MMAs of n - stages.
        after["fetch", n] = [("seen", n - stages, (n - stages) & 7)] if n >= stages else []
        after["split", n] = [("fetch", n)]  # writes the scales
        after["mma", n] = [("split", n)] + [("freed", n - buffers, w) for w in range(warps) if n >= buffers]
        for w in range(warps):
            after["seen", n, w] = [("mma", n)] + [("read", n - 1, w)] * (n > 0)
            after["freed", n, w] = [("seen", n, w)]  # TMEM is read, the scales may not be
            after["read", n, w] = [("freed", n, w)]
    for n in range(slots, slabs):
        before, todo = set(), [("split", n)]
        while todo:
            for e in after[todo.pop()]:
                if e not in before:
                    before.add(e)
                    todo.append(e)
        assert all(("read", n - slots, w) in before for w in range(warps)), n
