"""The operators around the bf16 / FP8 linears on the GPU against plain 64-bit implementations.

Tolerances (bf16 rounds by at most 2^-8 of the value, E4M3 by 2^-4, or half its subnormal step 2^-9):

* norm: a row of d values sums its squares in fp32 with at most 64 + 13 additions in a chain
  (each 2^-24, halved by the square root), and makes six more roundings: under 2^-17 of the value;
* product: the accumulator adds one partial sum per 16 values of K; every addition, in the tensor
  core or after it, is taken as a full fp32 ulp (2^-23) of the largest partial sum, for which
  sum |x w| stands: (k / 16 + 64) 2^-23 sum |x w|.  The activations change a value by at most 1.13
  times its argument's change, and evaluate to 2^-17 of |z|.
"""
import math

import pytest
import torch

import flashvsr_optimizations_b200 as fvq
from flashvsr_optimizations_b200 import ops
from helpers import calls_with_a_tangent

pytestmark = pytest.mark.gpu

BF16, F32, F8, F64 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.float64
HALF_BF16, HALF_E4M3 = 2.0 ** -8, 2.0 ** -4


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, std=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * std).to(dtype)


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert ops.read_device_error() == 0


def inside(got, want, bound):
    """|got - want| <= bound everywhere, with the same NaN and infinities."""
    got, want = got.double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    over = ((got - want).abs() - bound)[fine]
    assert over.numel() == 0 or over.max().item() <= 0, f"exceeds the bound by {over.max().item():.3e}"


def codes_inside(q, scale, v, extra):
    """q are E4M3 codes of v / scale up to `extra` (relative) and half a step."""
    t = v / scale.double()
    inside(q.float(), t, torch.maximum(t.abs() * HALF_E4M3, torch.full_like(t, 2.0 ** -10)) + t.abs() * extra)


# ---------------------------------------------------------------- norm
def norm64(x, r, w, eps):
    s = x.double() if r is None else x.double() + r.double()
    v = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return s, v if w is None else v * w.double()


def check_norm(x, r, w, eps=1e-6):
    s, v = norm64(x, r, w, eps)
    tol = 2.0 ** -17
    if r is None:
        y = ops.rms_norm(x, w, eps)
        q, scale = ops.rms_norm_fp8(x, w, eps)
    else:
        y, new = ops.add_rms_norm(x, r, w, eps)
        q, scale, new2 = ops.add_rms_norm_fp8(x, r, w, eps)
        assert new.dtype == r.dtype and torch.equal(new, new2)
        want = (x.float() + r.float()).to(r.dtype)     # one fp32 addition, one rounding
        assert torch.equal(new, want)
    assert y.dtype == BF16 and y.shape == x.shape and q.dtype == F8 and scale.shape == (*x.shape[:-1], 1)
    inside(y, v, v.abs() * (HALF_BF16 + tol))
    want = (v.abs().amax(-1, keepdim=True) / 448).clamp_min(1e-12)
    inside(scale, want, want * tol)
    codes_inside(q, scale, v, tol)


@pytest.mark.parametrize("d", [1, 2, 7, 8, 24, 64, 72, 127, 128, 129, 256, 264, 500, 512, 1000, 1024, 1536, 1544,
                               2040, 2047, 2048, 2049, 4096, 4104, 6000, 8192, 8960, 10240, 12288, 12296, 16384])
@pytest.mark.parametrize("residual", [None, BF16, F32])
def test_norm_row_lengths(d, residual):
    rows = 37 if d < 2048 else 5
    x, w = randn(rows, d, seed=d), randn(d, seed=d + 1)
    r = None if residual is None else randn(rows, d, seed=d + 2, std=2.0, dtype=residual)
    check_norm(x, r, w)


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 33, 1000])
@pytest.mark.parametrize("d", [64, 128, 1536, 4096])
def test_norm_row_counts_and_no_weight(rows, d):
    check_norm(randn(rows, d, seed=rows), randn(rows, d, seed=rows + 1), None)
    check_norm(randn(rows, d, seed=rows), None, randn(d, seed=3), eps=0.0)


@pytest.mark.parametrize("d", [128, 80, 33])
def test_norm_strided_views(d):
    qkv = randn(50, 3 * 6 * d + 8, seed=d)
    heads = qkv[:, 6 * d:12 * d].unflatten(1, (6, d))           # [tokens, heads, d] inside wider rows
    w = randn(d, seed=1)
    check_norm(heads, None, w)
    check_norm(heads, randn(50, 6, d, seed=2), w)
    check_norm(qkv[:, 5:5 + d], None, w)                          # two-dimensional, odd offset
    check_norm(qkv[::2, :d], None, w)
    check_norm(heads.transpose(0, 1), None, w)
    check_norm(qkv[:12, :d].view(2, 2, 3, d).transpose(0, 2), None, w)   # four dimensions: copied
    check_norm(qkv[:1, :d].expand(9, d), None, w)                 # broadcast rows
    check_norm(qkv[0, :d], None, w)                               # a single vector
    check_norm(qkv[:4, :d].t(), None, None)                       # no adjacent values: copied


@pytest.mark.parametrize("rows,d", [(9600, 264), (9600, 520), (4737, 515), (5001, 1536), (4800, 2047), (4740, 2048), (2400, 2050), (2400, 4096),
                                    (1300, 5555), (1250, 8960), (650, 12288), (700, 16384), (4737, 301)])
@pytest.mark.parametrize("residual", [None, BF16, F32])
def test_norm_many_rows(rows, d, residual):
    """Enough rows for the streaming form, from storage whose ends are the rows' ends."""
    x = randn(rows, d, seed=d)
    r = None if residual is None else randn(rows, d, seed=d + 1, dtype=residual)
    check_norm(x, r, randn(d, seed=d + 2))
    if d < 3000:
        check_norm(x[:, 1:], None if r is None else r[:, 1:], None)
        check_norm(x.view(-1)[3:3 + (rows - 1) * d].view(rows - 1, d), None, randn(d, seed=d + 3))


def test_norm_many_strided_rows():
    wide = randn(800, 6 * 512 + 24, seed=3)
    check_norm(wide[:, 8:8 + 6 * 512].unflatten(1, (6, 512)), None, randn(512, seed=4))
    check_norm(wide[:, 5:5 + 6 * 501].unflatten(1, (6, 501)), randn(800, 6, 501, seed=6), randn(501, seed=4))
    heads = randn(30000, 3 * 256, seed=5)
    check_norm(heads[:, 256:].unflatten(1, (4, 128)), None, randn(128, seed=4))
    check_norm(heads[:, 256:].unflatten(1, (8, 64)), randn(30000, 8, 64, seed=6, dtype=F32), randn(64, seed=4))
    check_norm(heads[:29999, 3:242], None, randn(239, seed=4))
    check_norm(wide[0, :300].expand(20000, 300), None, None)


def test_norm_wait_limit():
    """Whether or not a wait runs out of a limit of one test, the rows are waited for."""
    x, w = randn(60000, 1536, seed=1), randn(1536, seed=2)
    want = ops.rms_norm(x, w)
    torch.cuda.synchronize()
    ops.set_wait_limit(1)
    try:
        y = ops.rms_norm(x, w)
        assert ops.read_device_error() in (0, 1)
    finally:
        ops.set_wait_limit(0)
    assert torch.equal(y, want) and torch.equal(ops.rms_norm(x, w), want)


def test_norm_special_rows():
    d = 1536
    x = randn(8, d, seed=4)
    x[0] = 0.0
    x[1, 5] = float("inf")
    x[2, 7] = float("nan")
    x[3] = 1e-30
    x[4, 9] = float("-inf")
    x[5] = 1e15
    x[6, ::2] = -0.0
    w = randn(d, seed=5)
    s, v = norm64(x, None, w, 1e-6)
    y = ops.rms_norm(x, w)
    inside(y, v, v.abs() * (HALF_BF16 + 2.0 ** -17))
    q, scale = ops.rms_norm_fp8(x, w)
    assert (q[0].float() == 0).all() and scale[0].item() == pytest.approx(1e-12, rel=1e-6)
    # an infinity makes one NaN, a NaN all: the maximum is NaN then, and with it every code
    assert torch.isnan(scale[[1, 2, 4]]).all() and torch.isnan(q[[1, 2, 4]].float()).all()
    ok = [3, 5, 6, 7]
    codes_inside(q[ok], scale[ok], v[ok], 2.0 ** -17)
    assert torch.isfinite(ops.rms_norm(x[:1], w, 1e-6)).all()


def test_norm_empty_and_refusals():
    w = randn(64, seed=1)
    assert ops.rms_norm(randn(0, 64), w).shape == (0, 64)
    q, s, new = ops.add_rms_norm_fp8(randn(0, 3, 64), randn(0, 3, 64), w)
    assert q.shape == (0, 3, 64) and s.shape == (0, 3, 1) and new.shape == (0, 3, 64)
    x = randn(4, 64)
    with pytest.raises(TypeError):
        ops.rms_norm(x.float(), w)
    with pytest.raises(ValueError):
        ops.rms_norm(x, w[:32])
    with pytest.raises(ValueError):
        ops.rms_norm(x, w.float())
    with pytest.raises(ValueError):
        ops.add_rms_norm(x, x[:2], w)
    with pytest.raises(ValueError):
        ops.add_rms_norm(x, x.half(), w)
    with pytest.raises(ValueError):
        ops.rms_norm(randn(4, 0), None)
    with pytest.raises(RuntimeError):
        ops.rms_norm(x, w.cpu())
    with pytest.raises(fvq.FvqError):
        ops.rms_norm(randn(2, 16385))
    with pytest.raises(fvq.FvqError):
        ops.rms_norm(x, w, -1.0)


# ---------------------------------------------------------------- product
ACT64 = {
    "none": lambda z: z,
    "relu": lambda z: torch.where(z < 0, torch.zeros_like(z), z),
    "gelu": lambda z: 0.5 * z * torch.special.erfc(-z / math.sqrt(2)),
    "gelu_tanh": lambda z: 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))),
    "silu": lambda z: z * torch.sigmoid(z),
}


def product64(x, w, sx, sw, bias, act, gated, residual):
    """(y, bound) of the formulas in 64 bits."""
    x2 = x.double().reshape(-1, x.shape[-1])
    w = w.double()
    z, mag = x2 @ w.t(), x2.abs() @ w.abs().t()
    if sx is not None:
        f = sx.double().reshape(-1, 1) * sw.double().reshape(1, -1)
        z, mag = z * f, mag * f
    if bias is not None:
        z, mag = z + bias.double(), mag + bias.double().abs()
    dz = (x.shape[-1] / 16 + 64) * 2.0 ** -23 * mag
    f = ACT64[act]
    if gated:
        n = w.shape[0] // 2
        h = f(z[:, :n]) * z[:, n:]
        dh = (1.13 * dz[:, :n] + 2.0 ** -17 * z[:, :n].abs()) * (z[:, n:].abs() + dz[:, n:]) \
            + f(z[:, :n]).abs() * dz[:, n:]
    else:
        h, dh = f(z), 1.13 * dz + 2.0 ** -17 * z.abs()
    if residual is not None:
        h = h + residual.double().reshape(h.shape)
    shape = (*x.shape[:-1], h.shape[1])
    return h.reshape(shape), (HALF_BF16 * h.abs() + (1 + HALF_BF16) * dh).reshape(shape)


def fp8_rows(rows, k, seed, std=1.0):
    """Codes and row scales; any will do, and the row quantizer ends at 16384 values."""
    x = randn(rows, k, seed=seed, std=std).float()
    scale = x.abs().amax(-1, keepdim=True) / 448
    return (x / scale).to(F8), scale


def check_product(m, n, k, fp8=False, bias=True, act="none", gated=False, residual=True, seed=0):
    wn = 2 * n if gated else n
    b = randn(wn, seed=seed + 2) if bias else None
    r = randn(m, n, seed=seed + 3) if residual else None
    std = 1 / math.sqrt(k)
    if fp8:
        x, sx = fp8_rows(m, k, seed)
        w, sw = fp8_rows(wn, k, seed + 1, std)
        y = ops.fp8_scaled_mm_act(x, sx, w, sw, b, act, gated, r)
        again = ops.fp8_scaled_mm_act(x, sx, w, sw, b, act, gated, r)
    else:
        x, w, sx, sw = randn(m, k, seed=seed), randn(wn, k, seed=seed + 1, std=std), None, None
        y = ops.linear_act(x, w, b, act, gated, r)
        again = ops.linear_act(x, w, b, act, gated, r)
    assert y.dtype == BF16 and y.shape == (m, n)
    assert torch.equal(y, again)
    want, bound = product64(x.float() if fp8 else x, w.float() if fp8 else w, sx, sw, b, act, gated, r)
    inside(y, want, bound)


@pytest.fixture(params=[1, 2], ids=["split", "pair"])
def kernel(request):
    ops.set_linear_kernel(request.param)
    yield request.param
    ops.set_linear_kernel(0)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 100, 128, 129, 256, 257, 300, 515])
def test_product_row_counts(kernel, fp8, m):
    check_product(m, 264, 192, fp8)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("n", [8, 16, 56, 64, 72, 128, 136, 192, 200, 256, 264, 520])
def test_product_column_counts(kernel, fp8, n):
    check_product(70, n, 128, fp8)
    check_product(70, n, 128, fp8, act="silu", gated=True, residual=False)


@pytest.mark.parametrize("k", [8, 16, 24, 56, 64, 72, 136, 320, 1536, 1544, 8960])
def test_product_depths_bf16(kernel, k):
    check_product(33, 72, k)


@pytest.mark.parametrize("k", [16, 48, 128, 144, 400, 1536, 1552, 8960])
def test_product_depths_fp8(kernel, k):
    check_product(33, 72, k, True)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
def test_product_epilogues(kernel, fp8, gated, act):
    for bias in (False, True):
        for residual in (False, True):
            check_product(150, 168, 96, fp8, bias, act, gated, residual, seed=11)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k,gated", [(1, 8960, 1536, False), (24, 1536, 8960, False), (129, 4104, 512, True),
                                         (777, 1536, 1536, True), (2500, 1536, 1024, False),
                                         (4096, 2304, 128, False), (1, 8, 16, False), (20000, 8, 64, False),
                                         (3, 20000, 64, True)])
def test_product_by_size(fp8, m, n, k, gated):
    check_product(m, n, k, fp8, act="gelu_tanh" if gated else "none", gated=gated)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("n,k", [(8, 16), (16, 528), (72, 1536), (1000, 8960), (8960, 1536), (264, 12288), (40, 20480)])
def test_product_few_rows(fp8, m, n, k):
    """One or two rows (the form that streams W past x), and the next counts."""
    check_product(m, n, k, fp8)
    check_product(m, n, k, fp8, act="gelu_tanh", gated=True, residual=False)
    check_product(m, n, k, fp8, bias=False, act="silu", gated=True)


@pytest.mark.parametrize("m", [1, 3])
def test_product_few_rows_views(m):
    wide = randn(m, 400, seed=1)
    w = randn(72, 128, seed=2)
    for x in (wide[:, 8:136], wide[:, 4:132], wide[:1, :128].expand(m, 128)):
        want, bound = product64(x, w, None, None, None, "silu", False, None)
        inside(ops.linear_act(x, w, act="silu"), want, bound)


def test_product_extreme_values(kernel):
    """Activations far out on both sides, infinities and NaN go where the formulas put them."""
    k, n, m = 64, 64, 40
    x = torch.zeros(m, k, dtype=BF16, device="cuda")
    z = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 3.0, -3.0, 20.0, -20.0, 88.0, -88.0, 100.0, -100.0, 1e4, -1e4,
                      1e13, -1e13, 1e30, -1e30, float("inf"), float("nan")], dtype=BF16, device="cuda")
    x[:20, 0] = z
    x[20:, 0] = z
    w = torch.zeros(n, k, dtype=BF16, device="cuda")
    w[:, 0] = 1.0
    # the other products of a row are 0 * 0, an infinity meets only its own 1
    for act in ops.ACTIVATIONS:
        y = ops.linear_act(x, w, act=act).double()
        zz = x[:, :1].double().expand(m, n)
        want = ACT64[act](zz)
        if act in ("gelu_tanh", "gelu", "silu"):
            want = torch.where(zz == float("inf"), zz, want)
        assert torch.equal(torch.isnan(y), torch.isnan(want)), act
        fine = torch.isfinite(want)
        assert torch.equal(y[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
        # 88 * 2^-23 from the exponent's argument; tails under the smallest normal may be flushed
        tol = want.abs() * (HALF_BF16 + 2.0 ** -15) + 2.0 ** -125
        assert ((y - want).abs() <= tol)[fine].all(), act


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_activations_of_every_bf16_between_2_to_minus_20_and_40(kernel, act, gated):
    """The relative error holds down both tails, not only where the values are large."""
    bits = torch.arange(0x3580, 0x4220, dtype=torch.int32, device="cuda")
    z = torch.cat([bits, bits | 0x8000]).to(torch.uint16).view(BF16)
    x = torch.zeros(z.numel(), 16, dtype=BF16, device="cuda")
    x[:, 0], x[:, 1] = z, 1.0
    w = torch.zeros(16 if gated else 8, 16, dtype=BF16, device="cuda")
    w[:8, 0] = 1.0
    if gated:
        w[8:, 1] = 1.0
    y = ops.linear_act(x, w, act=act, gated=gated).double()
    # 1 + tanh(t) is 2 sigmoid(2 t); the former loses the tail's digits in 64 bits too
    f = (lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))) \
        if act == "gelu_tanh" else ACT64[act]
    want = f(z.double())[:, None].expand_as(y)
    # the exponent's argument is at most 126 (in powers of two) where the result is not flushed and
    # is rounded six times, constants included: 6 * 126 * ln 2 * 2^-24 < 2^-14.9; the exponential,
    # the reciprocal and the products beside it add less than 2^-19
    assert ((y - want).abs() <= want.abs() * (HALF_BF16 + 2.0 ** -14.8) + 2.0 ** -125).all()


def test_product_views_and_leading_dimensions(kernel):
    wide = randn(2, 40, 400, seed=1)
    w = randn(72, 128, seed=2)
    cases = [wide[0, :, 8:136], wide[0, :, 4:132], wide[0, ::2, 16:144], wide[:, :, :128],
             wide[:, :, 200:328].transpose(0, 1), wide[0, 0, :128], wide[0, :1, :128].expand(9, 128),
             wide[0, :1, 8:136]]
    for x in cases:
        r = randn(*x.shape[:-1], 72, seed=3)
        y = ops.linear_act(x, w, act="silu", residual=r)
        want, bound = product64(x, w, None, None, None, "silu", False, r)
        inside(y, want, bound)
    q, s = ops.fp8_row_quant(randn(40, 400, seed=4))
    wq, ws = ops.fp8_row_quant(w)
    for x in (q[:, 16:144], q[:, 8:136], q[::3, :128]):
        sx = s[::3] if x.shape[0] != 40 else s
        y = ops.fp8_scaled_mm_act(x, sx, wq, ws.flatten())
        want, bound = product64(x.float(), wq.float(), sx, ws, None, "none", False, None)
        inside(y, want, bound)
    off = randn(73 * 128 + 4, seed=5)[4:4 + 72 * 128].view(72, 128)     # weight at 8 bytes past alignment
    y = ops.linear_act(wide[0, :, :128], off, bias=randn(73, seed=6)[1:])
    want, bound = product64(wide[0, :, :128], off, None, None, randn(73, seed=6)[1:], "none", False, None)
    inside(y, want, bound)


def test_product_rows_do_not_see_one_another(kernel):
    """A NaN row of x, a NaN row of W and a NaN residual stay where they are."""
    m, n, k = 140, 136, 256
    x, w, r = randn(m, k, seed=1), randn(n, k, seed=2), randn(m, n, seed=3)
    clean = ops.linear_act(x, w, residual=r)
    x[17], w[33], r[50, 60] = float("nan"), float("nan"), float("nan")
    y = ops.linear_act(x, w, residual=r)
    hit = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    hit[17], hit[:, 33], hit[50, 60] = True, True, True
    assert torch.equal(torch.isnan(y), hit) and torch.equal(y[~hit], clean[~hit])


@pytest.mark.parametrize("m,n,k,gated", [(24, 264, 1536, False), (600, 520, 4096, True), (2000, 1536, 512, False)])
def test_product_wait_limit(kernel, m, n, k, gated):
    """With a limit of one test per wait the kernels give up, drain and report; the next call is right."""
    wn = 2 * n if gated else n
    x, w, r = randn(m, k, seed=1), randn(wn, k, seed=2, std=k ** -0.5), randn(m, n, seed=3)
    want = ops.linear_act(x, w, act="silu", gated=gated, residual=r)
    assert ops.read_device_error() == 0
    ops.set_wait_limit(1)
    try:
        ops.linear_act(x, w, act="silu", gated=gated, residual=r)
        assert ops.read_device_error() != 0
    finally:
        ops.set_wait_limit(0)
    assert torch.equal(ops.linear_act(x, w, act="silu", gated=gated, residual=r), want)


def test_product_empty_and_refusals():
    x, w = randn(4, 64), randn(72, 64)
    assert ops.linear_act(x[:0], w).shape == (0, 72)
    assert ops.linear_act(randn(2, 0, 64), w, act="silu", gated=True).shape == (2, 0, 36)
    assert ops.linear_act(x, w[:0]).shape == (4, 0)
    q, s = ops.fp8_row_quant(x)
    wq, ws = ops.fp8_row_quant(w)
    for bad, kind in ((lambda: ops.linear_act(x.float(), w), TypeError),
                      (lambda: ops.linear_act(x, w.float()), TypeError),
                      (lambda: ops.linear_act(x, w[:, :56]), ValueError),
                      (lambda: ops.linear_act(x, w[:71], gated=True), ValueError),
                      (lambda: ops.linear_act(x, w, act="tanh"), ValueError),
                      (lambda: ops.linear_act(x, w, bias=x[0]), ValueError),
                      (lambda: ops.linear_act(x, w, residual=x), ValueError),
                      (lambda: ops.linear_act(x, w, residual=randn(4, 72).float()), ValueError),
                      (lambda: ops.linear_act(x, w.cpu()), RuntimeError),
                      (lambda: ops.linear_act(x, w[:71]), fvq.FvqError),            # n % 8
                      (lambda: ops.linear_act(x[:, :60], w[:, :60]), fvq.FvqError),  # k % 8
                      (lambda: ops.fp8_scaled_mm_act(x, s, wq, ws), TypeError),
                      (lambda: ops.fp8_scaled_mm_act(q, s[:3], wq, ws), ValueError),
                      (lambda: ops.fp8_scaled_mm_act(q, s.double(), wq, ws), ValueError),
                      (lambda: ops.fp8_scaled_mm_act(q[:, :56], s, wq[:, :56], ws), fvq.FvqError)):
        with pytest.raises(kind):
            bad()


def test_no_gradient():
    x, w = randn(4, 64), randn(72, 64).requires_grad_()
    y = ops.linear_act(x, w)
    with pytest.raises(RuntimeError, match="no gradient formula"):
        y.float().sum().backward()
    with torch.no_grad():
        assert not ops.linear_act(x, w).requires_grad
    y, s = ops.add_rms_norm(x.requires_grad_(), x.detach())
    with pytest.raises(RuntimeError, match="no gradient formula"):
        s.float().sum().backward()


# ---------------------------------------------------------------- paged FP8 keys and values
def store(pages, page, heads, d, seed=0):
    codes = [randn(pages, page, heads, d, seed=seed + i).to(F8) for i in (0, 1)]
    scales = [torch.rand(pages, page, heads, generator=gen(seed + 5 + i), device="cuda") + 0.5 for i in (0, 1)]
    return codes[0], scales[0], codes[1], scales[1]


def row_scale(x):
    return torch.maximum(x.float().abs().amax(-1) / torch.tensor(448.0, device=x.device),
                         torch.tensor(1e-12, device=x.device))


def check_written(x, slots, codes, scale, before_codes, before_scale):
    codes, scale = codes.flatten(0, 1), scale.flatten(0, 1)
    kept = torch.ones(codes.shape[0], dtype=torch.bool, device="cuda")
    live = (slots >= 0) & (slots < codes.shape[0])
    kept[slots[live]] = False
    assert torch.equal(codes.view(torch.uint8)[kept], before_codes.view(torch.uint8).flatten(0, 1)[kept])
    assert torch.equal(scale[kept], before_scale.flatten(0, 1)[kept])
    got, x = scale[slots[live]], x[live]
    assert torch.equal(got, row_scale(x))                    # an exact maximum and one IEEE division
    # x * (1 / scale): two roundings of 2^-24 before E4M3's
    codes_inside(codes[slots[live]], got[..., None], x.double(), 2.0 ** -22)


@pytest.mark.parametrize("tokens", [1, 2, 3, 40, 300])
@pytest.mark.parametrize("heads,d,page", [(1, 8, 1), (12, 128, 16), (5, 64, 48), (3, 80, 16), (2, 256, 64), (7, 264, 5),
                                          (2, 512, 16)])
def test_cache_write(tokens, heads, d, page):
    pages = (tokens + page - 1) // page + 2
    cache = store(pages, page, heads, d)
    before = [t.clone() for t in cache]
    qkv = randn(tokens, 3, heads, d, seed=7)
    qkv[0, :, 0] = 0.0                                      # a row of zeros: the smallest scale
    slots = torch.randperm(pages * page, generator=gen(1), device="cuda")[:tokens]
    if tokens > 2:
        slots[1], slots[tokens - 1] = -1, -7
    ops.fp8_cache_write(qkv[:, 1], qkv[:, 2], slots, *cache)
    check_written(qkv[:, 1], slots, cache[0], cache[1], before[0], before[1])
    check_written(qkv[:, 2], slots, cache[2], cache[3], before[2], before[3])


def test_cache_write_views_special_values_and_bad_slots():
    heads, d = 4, 64
    cache = store(4, 16, heads, d)
    before = [t.clone() for t in cache]
    base = randn(heads, 30, d + 8, seed=3)
    k = base[:, :, :d].transpose(0, 1)                       # heads outermost
    v = base[:, :, 4:4 + d].transpose(0, 1)                  # off 16 bytes: copied
    slots = torch.randperm(64, generator=gen(2), device="cuda")[:30]
    slots[3], slots[4] = 64, 1 << 40                         # past the store: skipped and reported
    ops.fp8_cache_write(k, v, slots, *cache)
    assert ops.read_device_error() == 64
    check_written(k, slots, cache[0], cache[1], before[0], before[1])
    check_written(v, slots, cache[2], cache[3], before[2], before[3])
    x = randn(3, heads, d, seed=4)
    x[0, 0, 1], x[1, 1, 2] = float("inf"), float("nan")
    ops.fp8_cache_write(x, x, torch.arange(3, device="cuda"), *cache)
    codes, scale = cache[0].flatten(0, 1).float(), cache[1].flatten(0, 1)
    assert scale[0, 0] == float("inf") and torch.isnan(codes[0, 0, 1]) and (codes[0, 0, 2:] == 0).all()
    assert torch.isnan(scale[1, 1]) and torch.isnan(codes[1, 1]).all()
    assert torch.isfinite(codes[2]).all() and torch.isfinite(codes[0, 1:]).all()


def read64(cache, table, lens, most):
    """bf16(q * scale) below the length, zero above; one fp32 product, one rounding: exact."""
    out = []
    page = cache[0].shape[1]
    for codes, scale in ((cache[0], cache[1]), (cache[2], cache[3])):
        full = codes.float() * scale[..., None]
        o = torch.zeros(len(lens), most, *codes.shape[2:], device="cuda")
        for b, n in enumerate(lens):
            n = min(max(n, 0), most, table.shape[1] * page)
            for p in range(n):
                at = int(table[b, p // page])
                if 0 <= at < codes.shape[0]:
                    o[b, p] = full[at, p % page]
        out.append(o.to(BF16))
    return out


@pytest.mark.parametrize("heads,d,page,lens,most", [(1, 8, 1, [0, 1, 3], 3), (12, 128, 16, [33, 0, 16, 17], 40),
                                                    (5, 80, 7, [1], 1), (2, 264, 48, [50, 48], 61),
                                                    (3, 512, 16, [15, 20], 20)])
def test_cache_read(heads, d, page, lens, most):
    per = -(-most // page)
    cache = store(per * len(lens) + 2, page, heads, d)
    table = torch.randperm(per * len(lens) + 2, generator=gen(3), device="cuda")[:per * len(lens)]
    table = table.view(len(lens), per).to(torch.int32)
    for b, n in enumerate(lens):                             # entries past a length are not read
        table[b, -(-n // page):] = 1 << 30
    k, v = ops.fp8_cache_read(*cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), most)
    want = read64(cache, table.cpu(), lens, most)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_cache_read_bad_pages_and_lengths():
    cache = store(6, 16, 2, 64)
    table = torch.tensor([[0, 1], [6, 2], [-1, 3], [4, 5]], dtype=torch.int32, device="cuda")
    lens = [20, 20, 20, 20]
    k, v = ops.fp8_cache_read(*cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 32)
    assert ops.read_device_error() == 128
    want = read64(cache, table.cpu(), lens, 32)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    good = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    for lens, most, bits in (([-5, 3], 32, 0), ([33, 3], 40, 128), ([12, 3], 10, 128), ([10, 3], 10, 0)):
        k, v = ops.fp8_cache_read(*cache, good, torch.tensor(lens, dtype=torch.int32, device="cuda"), most)
        assert ops.read_device_error() == bits
        want = read64(cache, good.cpu(), lens, most)
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_cache_empty_and_refusals():
    cache = store(2, 16, 2, 64)
    before = [t.clone() for t in cache]
    kv, slots = randn(3, 2, 64), torch.arange(3, device="cuda")
    ops.fp8_cache_write(kv[:0], kv[:0], slots[:0], *cache)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, before))
    table, lens = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    assert ops.fp8_cache_read(*cache, table, lens, 0)[0].shape == (2, 0, 2, 64)
    assert ops.fp8_cache_read(*cache, table[:0], lens[:0], 5)[1].shape == (0, 5, 2, 64)
    for bad, kind in ((lambda: ops.fp8_cache_write(kv.float(), kv, slots, *cache), TypeError),
                      (lambda: ops.fp8_cache_write(kv, kv[:2], slots, *cache), ValueError),
                      (lambda: ops.fp8_cache_write(kv[:, :1], kv[:, :1], slots, *cache), ValueError),
                      (lambda: ops.fp8_cache_write(kv, kv, slots.int(), *cache), ValueError),
                      (lambda: ops.fp8_cache_write(kv, kv, slots[:2], *cache), ValueError),
                      (lambda: ops.fp8_cache_write(kv, kv, slots.cpu(), *cache), RuntimeError),
                      (lambda: ops.fp8_cache_write(kv, kv, slots, cache[0][:, ::2], cache[1][:, ::2],
                                                   cache[2][:, ::2], cache[3][:, ::2]), ValueError),
                      (lambda: ops.fp8_cache_read(*cache, table.long(), lens, 4), ValueError),
                      (lambda: ops.fp8_cache_read(*cache, table, lens[:1], 4), ValueError),
                      (lambda: ops.fp8_cache_read(*cache, table, lens, -1), ValueError),
                      (lambda: ops.fp8_cache_read(*cache, table[:, :0], lens, 4), ValueError),
                      (lambda: ops.fp8_cache_read(cache[0], cache[1].double(), cache[2], cache[3], table, lens, 4),
                       ValueError)):
        with pytest.raises(kind):
            bad()


# ---------------------------------------------------------------- streams and graphs
def block_inputs(m, seed):
    d, f, heads = 256, 512, 2
    return {"x": randn(m, d, seed=seed), "r": randn(m, d, seed=seed + 1), "slots": torch.arange(m, device="cuda") * 2}


def block_weights():
    d, f = 256, 512
    quant = lambda n, k, seed: ops.fp8_row_quant(randn(n, k, seed=seed, std=k ** -0.5))  # noqa: E731
    return {"norm": randn(d, seed=50), "qkv": quant(3 * d, d, 51), "o": quant(d, d, 52), "up": quant(2 * f, d, 53),
            "down": quant(d, f, 54), "bias": randn(d, seed=55)}


def run_block(i, w, cache, table, lens, most):
    """norm -> product -> store -> read -> attention in torch -> product + residual -> norm ->
    gated product -> product + residual: the operators as a block uses them."""
    d, heads = 256, 2
    q, s, r = ops.add_rms_norm_fp8(i["x"], i["r"], w["norm"])
    qkv = ops.fp8_scaled_mm_act(q, s, *w["qkv"]).unflatten(1, (3, heads, d // heads))
    ops.fp8_cache_write(qkv[:, 1], qkv[:, 2], i["slots"], *cache)
    k, v = ops.fp8_cache_read(*cache, table, lens, most)
    p = torch.softmax(torch.einsum("mhd,lhd->hml", qkv[:, 0].float(), k[0].float()) * (d // heads) ** -0.5, -1)
    att = torch.einsum("hml,lhd->mhd", p, v[0].float()).flatten(1).to(BF16)
    r = ops.fp8_scaled_mm_act(*ops.fp8_row_quant(att), *w["o"], residual=r)
    h = ops.fp8_scaled_mm_act(*ops.rms_norm_fp8(r, w["norm"]), *w["up"], act="silu", gated=True)
    return ops.fp8_scaled_mm_act(*ops.fp8_row_quant(h), *w["down"], w["bias"], residual=r)


def plain_block(i, w):
    """run_block in 64 bits on the dequantized weights, nothing else quantized."""
    d, heads = 256, 2
    full = {n: w[n][0].double() * w[n][1].double() for n in ("qkv", "o", "up", "down")}
    r, u = norm64(i["x"], i["r"], w["norm"], 1e-6)
    qkv = (u @ full["qkv"].t()).unflatten(1, (3, heads, d // heads))
    p = torch.softmax(torch.einsum("mhd,lhd->hml", qkv[:, 0], qkv[:, 1]) * (d // heads) ** -0.5, -1)
    r = r + torch.einsum("hml,lhd->mhd", p, qkv[:, 2]).flatten(1) @ full["o"].t()
    a, b = (norm64(r, None, w["norm"], 1e-6)[1] @ full["up"].t()).chunk(2, -1)
    return r + (a * torch.sigmoid(a) * b) @ full["down"].t() + w["bias"].double()


def fresh_store(m):
    cache = store(m, 2, 2, 128)
    table = torch.arange(m, dtype=torch.int32, device="cuda").view(1, m)
    return cache, table


@pytest.mark.parametrize("m", [1, 40, 300])
def test_block_run(m):
    """Frobenius-relative: every E4M3 rounding is at most 2^-4 (rms 2^-4 / sqrt(3) of the value,
    under 0.036) and independent; a branch passes at most five of them (norm, weight is exact,
    keys, values, attention output, gated product), so the output, which also carries the exact
    stream, is off by less than 0.036 * sqrt(5) < 0.09."""
    w, i = block_weights(), block_inputs(m, 60)
    cache, _ = fresh_store(2 * m)
    # slots 0, 2, 4, ...: one token per two-slot page is stored at its first slot
    i["slots"] = torch.randperm(4 * m, generator=gen(9), device="cuda")[:m]
    flat = [t.view(4 * m, 1, *t.shape[2:]) for t in cache]    # the same store as pages of one slot
    table = i["slots"].to(torch.int32).view(1, m)
    y = run_block(i, w, flat, table, torch.tensor([m], dtype=torch.int32, device="cuda"), m)
    want = plain_block(i, w)
    assert ((y.double() - want).norm() / want.norm()).item() < 0.09


def test_block_run_in_a_graph_and_on_streams():
    """The captured run replays with new inputs, two graphs and a side stream included."""
    m, w = 24, block_weights()
    lens = torch.tensor([m], dtype=torch.int32, device="cuda")

    def make(seed):
        i = block_inputs(m, seed)
        i["slots"] = torch.randperm(2 * m, generator=gen(seed), device="cuda")[:m]
        cache = store(2 * m, 1, 2, 128, seed=seed)
        return i, cache, i["slots"].to(torch.int32).view(1, m)

    want = {}
    for seed in (1, 2, 3):
        i, cache, table = make(seed)
        want[seed] = run_block(i, w, cache, table, lens, m)
    sets, graphs, outs = [make(1), make(2)], [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i, cache, table in sets:
            run_block(i, w, cache, table, lens, m)
    torch.cuda.current_stream().wait_stream(side)
    for i, cache, table in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run_block(i, w, cache, table, lens, m))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):                                     # both at once
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[1]) and torch.equal(outs[1], want[2])
    third, _, _ = make(3)
    sets[0][0]["x"].copy_(third["x"])
    sets[0][0]["r"].copy_(third["r"])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[3])                   # the slots differ, the attention does not see them


@pytest.mark.parametrize("m", [1, 24, 300])
def test_captured_between_copies_fills_and_a_second_stream(m):
    """Copies, fills, torch's kernels and events around the operators, captured and eager alike."""
    ws = [randn(256, 256, seed=s, std=1 / 16) for s in range(2)]
    x, w, one = randn(m, 256, seed=5), torch.empty_like(ws[0]), randn(256, seed=6)
    acc, side = torch.empty(m, 256, dtype=BF16, device="cuda"), torch.cuda.Stream()

    def chain():
        out = []
        for i in range(4):
            w.copy_(ws[i % 2])                      # a copy node
            acc.zero_()                             # a fill node
            y = ops.linear_act(x, w, act="silu", residual=acc)
            y.add_(1)                               # a kernel of torch's
            u = ops.rms_norm(y, one)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                v = ops.linear_act(u, w, act="relu")
            z = ops.linear_act(u, w, act="gelu")
            torch.cuda.current_stream().wait_stream(side)
            out.append(ops.add_rms_norm(z, v, one)[1])
        return out

    want = [t.clone() for t in chain()]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = chain()
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# ---------------------------------------------------------------- modules
def linear(out_f, in_f, seed, bias=True):
    lin = torch.nn.Linear(in_f, out_f, bias=bias, device="cuda", dtype=BF16)
    with torch.no_grad():
        lin.weight.copy_(randn(out_f, in_f, seed=seed, std=in_f ** -0.5))
        if bias:
            lin.bias.copy_(randn(out_f, seed=seed + 1, std=0.1))
    return lin


@pytest.mark.parametrize("shape", [(1, 512), (37, 512), (2, 150, 512), (0, 512)])
def test_fp8_ffn_prenorm(shape):
    """x + FFN(norm(x)) by the fused step: against its own launches one by one (the same bits), and
    against 64 bits on the dequantized weights (three E4M3 roundings on the branch's path, each
    at most 2^-4, rms 0.036: under 0.07 of the branch)."""
    ffn = fvq.FP8FFN(fvq.QuantLinear(linear(1024, 512, 1), "fp8"), torch.nn.GELU(approximate="tanh"),
                     fvq.QuantLinear(linear(512, 1024, 3), "fp8"))
    x, w = randn(*shape, seed=5), randn(512, seed=6)
    y = ffn.prenorm(x, w)
    assert y.shape == x.shape and y.dtype == BF16
    if not x.numel():
        return
    x2 = x.reshape(-1, 512)
    branch = ops.fp8_scaled_mm_act(*ops.rms_norm_fp8(x2, w), ffn[0].qweight, ffn[0].scale, ffn[0].bias, "gelu_tanh")
    again = ops.fp8_scaled_mm_act(*ops.fp8_row_quant(branch), ffn[2].qweight, ffn[2].scale, ffn[2].bias, residual=x2)
    assert torch.equal(y, again.reshape(shape))
    w1, w2 = (lin.qweight.double() * lin.scale.double() for lin in (ffn[0], ffn[2]))
    h = ACT64["gelu_tanh"](norm64(x2, None, w, 1e-6)[1] @ w1.t() + ffn[0].bias.double())
    want = h @ w2.t() + ffn[2].bias.double()
    got = y.reshape(-1, 512).double() - x2.double()
    # the output's own rounding, half a bf16 step of the sum, is counted apart
    slack = HALF_BF16 * (want + x2.double()).norm()
    assert (got - want).norm() <= 0.07 * want.norm() + slack
    with pytest.raises(ValueError):
        fvq.FP8FFN(ffn[0], torch.nn.GELU(), ffn[2]).prenorm(x, w)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_fp8_gated_ffn(act, bias):
    d, f = 256, 784
    gate, up, down = linear(f, d, 1, bias), linear(f, d, 3, bias), linear(d, f, 5, bias)
    ffn = fvq.FP8GatedFFN(gate, up, down, act)
    x, r, w = randn(3, 50, d, seed=7), randn(3, 50, d, seed=8), randn(d, seed=9)

    def branch(u):
        wg, wd = ffn.qweight.double() * ffn.scale.double(), ffn.down_qweight.double() * ffn.down_scale.double()
        z = u @ wg.t() + (0 if ffn.bias is None else ffn.bias.double())
        h = ACT64[act](z[:, :f]) * z[:, f:]
        return h @ wd.t() + (0 if ffn.down_bias is None else ffn.down_bias.double())

    x2 = x.reshape(-1, d).double()
    # x, and h from two products of x's roundings, and h's own: under 4 * 0.036 in all
    want = branch(x2)
    assert (ffn(x).reshape(-1, d).double() - want).norm() <= 0.15 * want.norm()
    for residual in (None, r):
        s, u = norm64(x, residual, w, 1e-6)
        want = branch(u.reshape(-1, d))
        got = ffn.prenorm(x, w, residual).reshape(-1, d).double() - s.reshape(-1, d)
        assert (got - want).norm() <= 0.15 * want.norm() + 2 * HALF_BF16 * (want + s.reshape(-1, d)).norm()
    assert set(ffn.state_dict()) >= {"qweight", "scale", "down_qweight", "down_scale"}


def test_kv_cache_object():
    heads, d, page = 3, 64, 16
    cache = fvq.FP8KVCache(10, page, heads, d)
    table = torch.tensor([[4, 2, 9], [7, 0, 1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([40, 19], dtype=torch.int32, device="cuda")
    at = torch.arange(40, device="cuda").repeat(2, 1)
    at[1, 19:] = -1                                         # the shorter sequence is padded
    kv = randn(2 * 40, 2, heads, d, seed=3)
    cache.write(kv[:, 0], kv[:, 1], cache.slots(table, at))
    k, v = cache.read(table, lens, 44)
    for got, x in ((k, kv[:, 0]), (v, kv[:, 1])):
        x = x.reshape(2, 40, heads, d)
        step = x.float().abs().amax(-1, keepdim=True) / 448
        for b, n in ((0, 40), (1, 19)):
            y, want = got[b, :n].double(), x[b, :n].double()
            # E4M3's half step (2^-10 of the scale below 2^-6), then bf16's
            bound = torch.maximum(want.abs() * HALF_E4M3, step[b, :n].double() * 2.0 ** -10)
            inside(y, want, bound * (1 + HALF_BF16) + HALF_BF16 * want.abs() + 2.0 ** -22 * want.abs())
            assert (got[b, n:] == 0).all()


@pytest.mark.parametrize("name", ["rms_norm", "add_rms_norm", "rms_norm_fp8", "add_rms_norm_fp8", "linear_act",
                                  "fp8_scaled_mm_act", "fp8_cache_write", "fp8_cache_read"])
def test_registered_operators(name):
    """Schemas (what is written in place, no aliases) and fake kernels, as torch checks them."""
    x, r, w = randn(6, 64, seed=1), randn(6, 64, seed=2, dtype=F32), randn(64, seed=3)
    q, s = ops.fp8_row_quant(x)
    wq, ws = ops.fp8_row_quant(randn(32, 64, seed=4))
    cache = store(3, 4, 2, 32)
    args = {"rms_norm": (x, w, 1e-6), "add_rms_norm": (x, r, w, 1e-6), "rms_norm_fp8": (x, None, 1e-6),
            "add_rms_norm_fp8": (x, r, w, 1e-6), "linear_act": (x, randn(32, 64, seed=5), None, "silu", True, None),
            "fp8_scaled_mm_act": (q, s, wq, ws, None, "none", False, randn(6, 32, seed=6)),
            "fp8_cache_write": (x.view(6, 2, 32), x.view(6, 2, 32), torch.arange(6, device="cuda"), *cache),
            "fp8_cache_read": (*cache, torch.zeros(1, 2, dtype=torch.int32, device="cuda"),
                               torch.ones(1, dtype=torch.int32, device="cuda"), 5)}[name]
    # torch's schema check multiplies its inputs, which E4M3 tensors do not do
    plain = not any(isinstance(a, torch.Tensor) and a.dtype == F8 for a in args)
    torch.library.opcheck(getattr(torch.ops.fvq, name).default, args,
                          test_utils=("test_schema", "test_faketensor") if plain else ("test_faketensor",))


def test_calls_that_the_short_path_leaves_to_python():
    """The same results through the registered operators and through the short path."""
    x, r, w = randn(40, 64, seed=1), randn(40, 64, seed=2), randn(64, seed=3)
    m, b = randn(72, 64, seed=4), randn(72, seed=5)
    op = torch.ops.fvq
    for a, c in zip(ops.add_rms_norm_fp8(x, r, w), op.add_rms_norm_fp8.default(x, r, w, 1e-6)):
        assert torch.equal(a.float(), c.float())
    assert torch.equal(ops.linear_act(x, m, b, "relu"), op.linear_act.default(x, m, b, "relu", False, None))
    q, s = ops.fp8_row_quant(x)
    wq, ws = ops.fp8_row_quant(m[:64])                        # gated: 32 columns
    assert torch.equal(ops.fp8_scaled_mm_act(q, s, wq, ws, act="silu", gated=True),
                       op.fp8_scaled_mm_act.default(q, s, wq, ws, None, "silu", True, None))
    c1, c2 = store(12, 4, 1, 64), store(12, 4, 1, 64)
    slots = torch.arange(40, device="cuda")
    ops.fp8_cache_write(x.view(40, 1, 64), r.view(40, 1, 64), slots, *c1)
    before = c1[0]._version
    ops.fp8_cache_write(x.view(40, 1, 64), r.view(40, 1, 64), slots, *c1)
    assert c1[0]._version > before                            # an in-place write is seen by autograd
    op.fp8_cache_write.default(x.view(40, 1, 64), r.view(40, 1, 64), slots, *c2)
    assert all(torch.equal(i.view(torch.uint8), j.view(torch.uint8)) for i, j in zip(c1, c2))
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(1, 12)
    lens = torch.tensor([40], dtype=torch.int32, device="cuda")
    for a, c in zip(ops.fp8_cache_read(*c1, table, lens, 44), op.fp8_cache_read.default(*c1, table, lens, 44)):
        assert torch.equal(a, c)


def test_other_threads_and_modes():
    """Calls from two threads on streams of their own, and under a dispatch mode."""
    import threading
    from torch.utils._python_dispatch import TorchDispatchMode
    x, w = randn(64, 512, seed=1), randn(256, 512, seed=2)
    want = ops.linear_act(x, w, act="silu")
    got = [None, None]

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got[i] = ops.linear_act(x, w, act="silu")
        s.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert torch.equal(got[0], want) and torch.equal(got[1], want)
    seen = []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    with Log():
        assert torch.equal(ops.linear_act(x, w, act="silu"), want)
    assert any("fvq.linear_act" in s for s in seen)
    with torch.inference_mode():
        assert torch.equal(ops.linear_act(x, w, act="silu"), want)
        cache = fvq.FP8KVCache(2, 4, 1, 64)
        kv = randn(3, 1, 64)
        cache.write(kv, kv, torch.arange(3, device="cuda"))
    with torch.no_grad():
        assert torch.equal(ops.linear_act(x, torch.nn.Parameter(w), act="silu"), want)


# ---------------------------------------------------------------- past 2^31 elements
def test_large_tensors():
    """Offsets that pass 32 bits: the last rows of tensors of 2.4e9 elements."""
    rows, d = 300_000, 8192
    x = torch.empty(rows, d, dtype=BF16, device="cuda")
    tail = randn(400, d, seed=1)
    x[-400:] = tail
    x[:400] = tail
    w = randn(d, seed=2)
    q, scale = ops.rms_norm_fp8(x, w)
    _, v = norm64(tail, None, w, 1e-6)
    for part in (slice(0, 400), slice(rows - 400, rows)):
        codes_inside(q[part], scale[part], v, 2.0 ** -17)
    del q, scale
    wide = x.view(rows * 64, 128)                              # short rows: the sub-warp form
    y = ops.rms_norm(wide)
    _, v = norm64(tail.view(-1, 128), None, None, 1e-6)
    inside(y[-400 * 64:], v, v.abs() * (HALF_BF16 + 2.0 ** -17))
    del y, wide, x
    torch.cuda.empty_cache()
    x, m = randn(rows, 64, seed=3), randn(d, 64, seed=4)
    r = torch.empty(rows, d, dtype=BF16, device="cuda")
    r[-400:] = tail
    y = ops.linear_act(x, m, act="silu", residual=r)
    want, bound = product64(x[-400:], m, None, None, None, "silu", False, tail)
    inside(y[-400:], want, bound)
    del y, r
    torch.cuda.empty_cache()


def test_large_store():
    """A store of 4.7e9 codes a side: slots and pages at its end."""
    pages, page, heads, d = 48_000, 64, 12, 128
    codes = [torch.empty(pages, page, heads, d, dtype=torch.uint8, device="cuda").view(F8) for _ in range(2)]
    scales = [torch.zeros(pages, page, heads, device="cuda") for _ in range(2)]
    cache = codes[0], scales[0], codes[1], scales[1]
    kv = randn(100, 2, heads, d, seed=1)
    table = torch.tensor([[pages - 1, pages - 3], [0, pages - 2]], dtype=torch.int32, device="cuda")
    at = torch.arange(100, device="cuda")
    slots = table[0].long()[at // page] * page + at % page
    ops.fp8_cache_write(kv[:, 0], kv[:, 1], slots, *cache)
    k, v = ops.fp8_cache_read(*cache, table, torch.tensor([100, 0], dtype=torch.int32, device="cuda"), 100)
    for got, x in ((k, kv[:, 0]), (v, kv[:, 1])):
        step = row_scale(x)[..., None].double()
        bound = torch.maximum(x.double().abs() * HALF_E4M3, step * 2.0 ** -10)
        inside(got[0], x.double(), bound * (1 + HALF_BF16) + (HALF_BF16 + 2.0 ** -22) * x.double().abs())
        assert (got[1] == 0).all()
    del codes, scales, cache
    torch.cuda.empty_cache()


def test_store_written_and_read_back_to_back():
    """Each kernel may start while the one before it runs; it reads what that one stored."""
    cache = fvq.FP8KVCache(24, 16, 4, 64)
    table = torch.randperm(24, device="cuda").to(torch.int32).reshape(2, 12)
    at = torch.arange(192, device="cuda").expand(2, 192)
    slots = cache.slots(table, at)
    lengths = torch.full((2,), 192, dtype=torch.int32, device="cuda")
    values = [randn(384, 4, 64, seed=s) for s in range(8)]
    got = []
    for i in range(64):
        cache.write(values[i % 8], values[(i + 3) % 8], slots)
        got.append(cache.read(table, lengths, 192))
    for i, (k, v) in enumerate(got):
        for y, x in ((k, values[i % 8]), (v, values[(i + 3) % 8])):
            if i < 8:
                inside(y.reshape(384, 4, 64), x.double(), (2.0 ** -4 + 2.0 ** -7) * x.double().abs()
                       + 2.0 ** -9 * x.double().abs().amax(-1, keepdim=True) / 448)
            else:
                assert torch.equal(y, got[i - 8][0 if y is k else 1])
    assert ops.read_device_error() == 0


@pytest.mark.parametrize("m", [1, 24])
def test_product_operands_written_just_before(m):
    """A weight that the kernel before wrote in place, over one that was just multiplied."""
    x = randn(m, 256, seed=1)
    ws = [randn(128, 256, seed=2 + i) for i in range(4)]
    w = torch.empty_like(ws[0])
    one = torch.ones(256, dtype=BF16, device="cuda")
    got = []
    for i in range(32):
        w.copy_(ws[i % 4])
        got.append(ops.linear_act(ops.linear_act(x, w), ws[0][:, :128].contiguous(), gated=1))
    for i in range(4, 32):
        assert torch.equal(got[i], got[i - 4])
    x2 = ops.rms_norm(x, one)
    assert torch.equal(ops.linear_act(x2, ws[1], gated=True), ops.linear_act(x2, ws[1], gated=1))


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m", [1, 2])
@pytest.mark.parametrize("n,k", [(8, 16384), (16, 16400), (80008, 16), (77000, 144), (1184, 1536), (2376, 8960),
                                 (9000, 512), (600, 4096), (5000, 400), (304, 2816), (40, 33024)])
def test_product_few_rows_shares_of_a_row(m, n, k, fp8):
    """One to eight warps a row, rings of few and many slots, several blocks a CTA, rows too long."""
    check_product(m, n, k, fp8, act="silu")
    check_product(m, n, k, fp8, act="silu", gated=True, residual=False)


def test_product_few_rows_nan_and_infinity_stay_in_their_row():
    x, w = randn(2, 528, seed=1), randn(1400, 528, seed=2)
    clean = ops.linear_act(x, w)
    w[33], w[34, 7], w[700] = float("nan"), float("inf"), float("nan")
    y = ops.linear_act(x, w)
    hit = torch.zeros(2, 1400, dtype=torch.bool, device="cuda")
    hit[:, 33], hit[:, 34], hit[:, 700] = True, True, True
    assert torch.equal(~torch.isfinite(y), hit) and torch.equal(y[~hit], clean[~hit])


@pytest.mark.parametrize("m,n,k,gated", [(1, 264, 1536, False), (2, 3000, 8960, True), (1, 80000, 64, False)])
def test_product_few_rows_wait_limit(m, n, k, gated):
    """A wait that runs out is reported; a copy that landed before its only test gives the result."""
    x, w = randn(m, k, seed=1), randn(2 * n if gated else n, k, seed=2, std=k ** -0.5)
    want = ops.linear_act(x, w, act="silu", gated=gated)
    ops.set_wait_limit(1)
    try:
        y = ops.linear_act(x, w, act="silu", gated=gated)
        assert ops.read_device_error() != 0 or torch.equal(y, want)
    finally:
        ops.set_wait_limit(0)
    assert torch.equal(ops.linear_act(x, w, act="silu", gated=gated), want)


# ---------------------------------------------------------------- under torch.jit.trace
@pytest.mark.parametrize("name", ["rms_norm", "add_rms_norm", "rms_norm_fp8", "add_rms_norm_fp8", "linear_act",
                                  "fp8_scaled_mm_act", "fp8_cache_write", "fp8_cache_read"])
def test_traced_with_one_input_and_run_with_another(name):
    """A trace records the operator, not the outputs it had while it was traced."""
    w, m = randn(64, seed=3), randn(32, 64, seed=4)
    mq, ms = ops.fp8_row_quant(m)
    slots = torch.arange(6, device="cuda")
    table, lens = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")

    def bits(t):
        return t.view(torch.uint8) if t.dtype == F8 else t

    def fresh(seed):
        x, r = randn(6, 64, seed=seed), randn(6, 64, seed=seed + 1)
        if name == "fp8_scaled_mm_act":
            return ops.fp8_row_quant(x)
        if name == "fp8_cache_write":
            return (x.view(6, 2, 32), r.view(6, 2, 32), *store(3, 4, 2, 32))
        return store(3, 4, 2, 32, seed=seed) if name == "fp8_cache_read" else (x, r)

    def write(k, v, *cache):
        ops.fp8_cache_write(k, v, slots, *cache)
        return cache

    fn = {"rms_norm": lambda x, r: ops.rms_norm(x, w) + r,
          "add_rms_norm": lambda x, r: ops.add_rms_norm(x, r, w),
          "rms_norm_fp8": lambda x, r: ops.rms_norm_fp8(x + r, w),
          "add_rms_norm_fp8": lambda x, r: ops.add_rms_norm_fp8(x, r, w),
          "linear_act": lambda x, r: ops.linear_act(x + r, m, act="silu"),
          "fp8_scaled_mm_act": lambda q, s: ops.fp8_scaled_mm_act(q, s, mq, ms),
          "fp8_cache_write": write,
          "fp8_cache_read": lambda *cache: ops.fp8_cache_read(*cache, table, lens, 5)}[name]
    traced = torch.jit.trace(fn, fresh(1), check_trace=False)
    want, got = fn(*fresh(11)), traced(*fresh(11))
    if isinstance(want, torch.Tensor):
        want, got = (want,), (got,)
    assert len(want) == len(got)
    for a, b in zip(want, got):
        assert torch.equal(bits(a), bits(b))


def test_traced_prenorm():
    ffn = fvq.FP8FFN(fvq.QuantLinear(linear(1024, 512, 1), "fp8"), torch.nn.GELU(approximate="tanh"),
                     fvq.QuantLinear(linear(512, 1024, 3), "fp8"))
    w = randn(512, seed=6)
    traced = torch.jit.trace(lambda x: ffn.prenorm(x, w), (randn(3, 512, seed=7),), check_trace=False)
    x = randn(3, 512, seed=8)
    assert torch.equal(traced(x), ffn.prenorm(x, w))


def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        for call in calls_with_a_tangent("cuda"):
            with pytest.raises(RuntimeError, match="no gradient formula"):
                call()
        x = randn(4, 64)
        assert torch.equal(ops.rms_norm(forward_ad.unpack_dual(forward_ad.make_dual(x, x)).primal), ops.rms_norm(x))


def test_tensors_without_memory_are_materialised():
    """A weight, bias or residual of zeros that torch holds without storage is not an absent one."""
    x, w = randn(8, 64, seed=1), randn(16, 64, seed=2)

    def zeros(*shape):
        return torch._efficientzerotensor(*shape, dtype=BF16, device="cuda")
    assert torch.equal(ops.rms_norm(x, zeros(64)), torch.zeros_like(x))
    assert torch.equal(ops.linear_act(x, w, zeros(16), residual=zeros(8, 16)), ops.linear_act(x, w))
    assert torch.equal(ops.linear_act(zeros(8, 64), w), torch.zeros(8, 16, dtype=BF16, device="cuda"))


def test_without_the_binding(monkeypatch):
    """The registered operators give the short path's results."""
    from flashvsr_optimizations_b200 import _lib
    x, r, w, m = randn(24, 64, seed=1), randn(24, 64, seed=2), randn(64, seed=3), randn(72, 64, seed=4)
    cache, slots = store(3, 16, 1, 64), torch.arange(24, device="cuda")
    table, lens = torch.arange(2, dtype=torch.int32, device="cuda").view(1, 2), torch.ones(1, dtype=torch.int32, device="cuda") * 24

    def run():
        y, s = ops.add_rms_norm(x, r, w)
        q, scale = ops.rms_norm_fp8(s, w)
        ops.fp8_cache_write(y.view(24, 1, 64), s.view(24, 1, 64), slots, *cache)
        return (y, s, q.view(torch.uint8), scale, ops.linear_act(y, m, act="silu"),
                ops.fp8_scaled_mm_act(q, scale, q, scale), *ops.fp8_cache_read(*cache, table, lens, 30))
    want = run()
    monkeypatch.setattr(_lib, "_binding", None)
    monkeypatch.setattr(_lib, "_binding_missing", True)
    for a, b in zip(want, run()):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- bf16 and E4M3 from one call of the C entry
# rows of 8, 16 and 32 lanes, with one and two rows a group; a CTA a row of 8 and of 16 values a thread; streamed by
# one to sixteen warps a row; each on and off 16 bytes
@pytest.mark.parametrize("rows,d", [(7, 33), (5, 64), (20000, 64), (9, 128), (40000, 121), (3, 256), (20000, 250), (6, 512),
                                    (20000, 511), (2, 1536), (3, 2047), (1, 16384), (5, 9001), (5001, 1536), (4800, 2047),
                                    (2400, 4096), (1200, 8200), (700, 16384), (700, 16383)])
@pytest.mark.parametrize("residual", [None, BF16, F32], ids=["none", "bf16", "fp32"])
def test_norm_with_both_outputs(rows, d, residual):
    from flashvsr_optimizations_b200 import _lib
    x, w = randn(rows, d, seed=1, std=2.0), randn(d, seed=2)
    r = None if residual is None else randn(rows, d, seed=3, dtype=residual)
    y, new = torch.empty_like(x), None if r is None else torch.empty_like(r)
    q, scale = torch.empty_like(x, dtype=F8), torch.empty(rows, 1, device="cuda")
    _lib.call("fvq_rms_norm", x.data_ptr(), rows, 1, d, 0, d, w.data_ptr(), 1e-6, None if r is None else r.data_ptr(),
              int(residual == F32), None if r is None else new.data_ptr(), y.data_ptr(), q.data_ptr(), scale.data_ptr(),
              torch.cuda.current_stream().cuda_stream)
    s, v = norm64(x, r, w, 1e-6)
    tol = 2.0 ** -17
    if r is not None:
        assert torch.equal(new, (x.float() + r.float()).to(residual))
    inside(y, v, v.abs() * (HALF_BF16 + tol))
    want = (v.abs().amax(-1, keepdim=True) / 448).clamp_min(1e-12)
    inside(scale, want, want * tol)
    codes_inside(q, scale, v, tol)


@pytest.mark.parametrize("limit", [1, 1000, 1500, 2000, 3000, 5000, 10000])
@pytest.mark.parametrize("m,n,k,gated", [(1, 264, 1536, False), (2, 3000, 8960, True), (1, 80000, 64, False),
                                         (1, 12288, 4096, False)])
def test_product_few_rows_right_whatever_the_wait_limit(m, n, k, gated, limit):
    """A wait that runs out is reported and waited for again before its slot is read: the result is right either way."""
    x, w = randn(m, k, seed=1), randn(2 * n if gated else n, k, seed=2, std=k ** -0.5)
    xq, wq = ops.fp8_row_quant(x), ops.fp8_row_quant(w)
    calls = (lambda: ops.linear_act(x, w, act="silu", gated=gated),
             lambda: ops.fp8_scaled_mm_act(*xq, *wq, act="silu", gated=gated))
    want = [call() for call in calls]
    ops.set_wait_limit(limit)
    try:
        for call, y in zip(calls, want):
            got = call()
            assert ops.read_device_error() in (0, 1)         # bit 0: a load's wait
            assert torch.equal(got, y)
    finally:
        ops.set_wait_limit(0)


def test_a_store_that_may_not_be_written_raises():
    """torch can mark a tensor's memory so that asking for a pointer to write throws."""
    cache = store(2, 4, 1, 64)
    x, slots = randn(3, 1, 64), torch.arange(3, device="cuda")
    torch._C._set_throw_on_mutable_data_ptr(cache[0])
    with pytest.raises(RuntimeError):
        ops.fp8_cache_write(x, x, slots, *cache)
    cache = store(2, 4, 1, 64)
    ops.fp8_cache_write(x, x, slots, *cache)                 # the interpreter goes on
