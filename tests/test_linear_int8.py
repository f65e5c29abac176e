"""8-bit linears (``ops.quantize_rows`` / ``ln_quantize_rows`` / ``linear_int8`` / ``ln_linear_int8``) against their
definitions in 64 bits, on the CPU reference and on the HIP kernels.

Tolerances.  quantize_rows: none (q is the correctly rounded quotient, scale one fp32 division).
linear_int8: the integer sum is exact; its conversion to fp32, two scale products and up to two additions round
5 times at 2^-24 of the largest magnitude, the activation adds at most 4e-7 of it (GELU: 1.5e-7 on erf, raw
exp2 / rcp 2^-22): 2^-20 of the magnitude covers both.  Then one rounding to the output type: half a step,
``finfo.eps / 2`` of the value (2^-25 in fp16's subnormals).
ln_quantize_rows: the fp32 LayerNorm is within 2^-17 of the row's largest value (two block sums of at most 2048
terms and five roundings), so q is within half a step plus 127 * 2^-17 of the 64-bit quotient."""
import math

import pytest
import torch
import torch.nn as nn

from arbius_amd import ops
from arbius_amd.models import layers

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32, device="cpu"):
    return torch.randn(*shape, generator=gen(seed)).to(dtype).to(device)


def quantize64(x):
    x = x.double()
    a = x.abs().amax(dim=-1, keepdim=True)
    q = torch.where(a > 0, torch.round(x * 127.0 / a), torch.zeros_like(x))
    return q, (a / 127.0)


def gelu64(x):
    return 0.5 * x * torch.special.erfc(-x / math.sqrt(2.0))


def linear64(q, sx, wq, sw, b, r, act):
    t = (q.double() @ wq.double().t()) * sx.double().reshape(-1, 1) * sw.double()
    y, mag = t, t.abs()
    for term in (b, r):
        if term is not None:
            y, mag = y + term.double(), mag + term.double().abs()
    if act == "gelu":
        y = gelu64(y)
    elif act == "quick_gelu":
        y = y * torch.sigmoid(1.702 * y)
    elif act == "geglu":
        h = y.shape[-1] // 2
        y, mag = y[:, :h] * gelu64(y[:, h:]), mag[:, :h] * mag[:, h:]
    return y, mag


def check(y, want, mag):
    half = torch.finfo(y.dtype).eps / 2
    err = (y.cpu().double().reshape(want.shape) - want).abs()
    over = err - (half * want.abs() + 2.0 ** -20 * mag + 2.0 ** -25)
    assert bool((over <= 0).all()), f"over the bound by {over.max().item():.3g}"


def rows(n, k, seed, device, dtype=torch.bfloat16):
    return ops.quantize_rows(randn(n, k, seed=seed, dtype=dtype, device=device) * (0.5 / math.sqrt(k)))


# ------------------------------------------------------------------ quantize_rows
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 16), (5, 77), (4, 320), (2, 2048), (7, 1101), (1, 20000), (300, 48)])
def test_quantize_rows_is_the_rounded_quotient(device, dtype, m, k):
    x = randn(m, k, seed=k, dtype=DTYPES[dtype], device=device)
    r = ops.quantize_rows(x)
    q, _ = quantize64(x.cpu())
    assert r.q.dtype == torch.int8 and torch.equal(r.q.cpu().double(), q)
    assert torch.equal(r.scale.cpu(), x.cpu().float().abs().amax(dim=1) / 127.0)
    assert r.shape == (m, k) and r.dtype == x.dtype


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_rows_half_steps_go_to_even(device, dtype):
    """Every row holds a = 127 * 2^e and the exact half steps (k + 1/2) 2^e and their neighbours."""
    dt = DTYPES[dtype]
    out = []
    for e in (0, -6, 5):
        v = torch.arange(-126, 127, dtype=torch.float64) + 0.5
        x = torch.cat([torch.tensor([127.0], dtype=torch.float64), v]) * 2.0 ** e
        out.append(x[:254])
    x = torch.stack(out).to(dt)
    x = torch.cat([x, torch.nextafter(x.float(), torch.full_like(x.float(), 1e9)).to(dt)])
    x[3:, 0] = x[:3, 0]
    r = ops.quantize_rows(x.to(device))
    q, _ = quantize64(x)
    assert torch.equal(r.q.cpu().double(), q)


@pytest.mark.parametrize("device", DEVICES)
def test_quantize_rows_extremes(device):
    big, tiny = torch.finfo(torch.bfloat16).max, 2.0 ** -130
    x = torch.zeros(7, 40)
    x[1] = torch.linspace(-1, 1, 40) * big
    x[2] = torch.linspace(-1, 1, 40) * tiny
    x[3, 5], x[4, 6], x[5, 39] = float("nan"), float("inf"), -float("inf")
    x[3:6, :4] = 1.0
    x[6, 7] = -2.0
    x = x.to(torch.bfloat16)
    r = ops.quantize_rows(x.to(device))
    q, _ = quantize64(x[[0, 1, 2, 6]])
    assert torch.equal(r.q.cpu()[[0, 1, 2, 6]].double(), q)
    assert r.scale[0] == 0 and r.scale.cpu()[3:6].isnan().all() and not bool(r.q[3:6].any())
    # what such a row yields: zeros (+ bias) and NaN
    w = rows(24, 40, 1, device)
    y = ops.linear_int8(x.to(device), w)
    assert not bool(y[0].any()) and bool(y[3:6].isnan().all()) and bool(y[[2, 6]].isfinite().all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantize_is_half_a_step_off(device, dtype):
    """Back in the tensor's shape and type: off by half a step of the row (scale / 2) and the type's own rounding, with
    2^-20 of the row's largest value for the scale's."""
    x = (randn(3, 5, 77, seed=1) * 4).to(DTYPES[dtype]).to(device)
    x[1, 2] = 0.0
    x[2, 4, 3] = float("inf")
    back = ops.quantize_rows(x).dequantize()
    assert back.shape == x.shape and back.dtype == x.dtype and bool(back[2, 4].isnan().all())
    assert not bool(back[1, 2].any())
    x, back = x.view(15, 77)[:14].double(), back.view(15, 77)[:14].double()
    top = x.abs().amax(dim=1, keepdim=True)
    half = torch.finfo(DTYPES[dtype]).eps / 2
    assert bool(((x - back).abs() <= top * (0.5 / 127 + 2.0 ** -20) * (1 + half) + half * x.abs()).all())


@pytest.mark.parametrize("device", DEVICES)
def test_quantize_rows_strided_views(device):
    base = randn(3, 5, 4, 96, seed=2, dtype=torch.bfloat16, device=device)
    for x in (base[:, :, 1], base[:, 2], base[1, :, :, 8:72], base[..., 3:80], base.transpose(0, 1), base[..., ::2],
              base[:1, :1, :1].expand(4, 1, 1, 96)):
        a, b = ops.quantize_rows(x), ops.quantize_rows(x.clone(memory_format=torch.contiguous_format))
        assert a.shape == tuple(x.shape) and torch.equal(a.q, b.q) and torch.equal(a.scale, b.scale)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 8), (5, 77), (3, 320), (4, 768), (2, 2048), (6, 1001), (130, 64)])
def test_ln_quantize_rows(device, dtype, m, k):
    dt = DTYPES[dtype]
    x = (randn(m, k, seed=3) * 3 + 0.5).to(dt)
    gamma, beta = (1 + 0.2 * randn(k, seed=4)).to(dt), (0.2 * randn(k, seed=5)).to(dt)
    r = ops.ln_quantize_rows(x.to(device), gamma.to(device), beta.to(device), 1e-5)
    x64 = x.double()
    y = (x64 - x64.mean(1, keepdim=True)) / torch.sqrt(x64.var(1, unbiased=False, keepdim=True) + 1e-5)
    y = y * gamma.double() + beta.double()
    a = y.abs().amax(dim=1, keepdim=True)
    assert bool(((r.scale.cpu().double()[:, None] * 127 / a - 1).abs() <= 2.0 ** -16).all())
    assert bool(((r.q.cpu().double() - 127 * y / a).abs() <= 0.5 + 127 * 2.0 ** -17).all())


# ------------------------------------------------------------------ linear_int8
SHAPES = [(1, 64, 64), (1, 16, 1), (1, 2048, 520), (2, 100, 30), (7, 1101, 33), (16, 640, 256), (17, 4096, 96),
          (33, 130, 257), (64, 128, 512), (100, 320, 960), (129, 1000, 200), (257, 768, 384), (300, 256, 1030),
          (513, 48, 130)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_int8_shapes(device, dtype, m, k, n):
    dt = DTYPES[dtype]
    x, w = randn(m, k, seed=m, dtype=dt, device=device), rows(n, k, n, device, dt)
    b, r = randn(n, seed=1, dtype=dt, device=device), randn(m, n, seed=2, dtype=dt, device=device)
    qx = ops.quantize_rows(x)
    for bias, res in ((None, None), (b, None), (b, r)):
        y = ops.linear_int8(x, w, bias, residual=res)
        assert y.dtype == dt and tuple(y.shape) == (m, n)
        cpu = [None if t is None else t.cpu() for t in (bias, res)]
        check(y, *linear64(qx.q.cpu(), qx.scale.cpu(), w.q.cpu(), w.scale.cpu(), *cpu, None))
    assert torch.equal(ops.linear_int8(qx, w, b, residual=r), ops.linear_int8(x, w, b, residual=r))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["gelu", "quick_gelu", "geglu"])
@pytest.mark.parametrize("m,k,n", [(1, 256, 512), (5, 77, 34), (40, 320, 640), (200, 128, 1034), (300, 640, 512)])
def test_linear_int8_activations(device, dtype, act, m, k, n):
    dt = DTYPES[dtype]
    x, w = (2 * randn(m, k, seed=m)).to(dt).to(device), ops.quantize_rows(
        randn(n, k, seed=n, dtype=dt, device=device) / math.sqrt(k))
    b = randn(n, seed=1, dtype=dt, device=device)
    qx = ops.quantize_rows(x)
    y = ops.linear_int8(x, w, b, act=act)
    check(y, *linear64(qx.q.cpu(), qx.scale.cpu(), w.q.cpu(), w.scale.cpu(), b.cpu(), None, act))
    if act != "geglu":
        r = randn(m, n, seed=2, dtype=dt, device=device)
        check(ops.linear_int8(x, w, b, residual=r, act=act),
              *linear64(qx.q.cpu(), qx.scale.cpu(), w.q.cpu(), w.scale.cpu(), b.cpu(), r.cpu(), act))


@pytest.mark.parametrize("device", DEVICES)
def test_linear_int8_full_scale_sums(device):
    """Every product 128 * 128 or -127 * 128: the largest sums, exact to the last bit before the scales."""
    for k in (16, 1000, 9001, ops.INT8_MAX_K):
        q = torch.full((3, k), -128, dtype=torch.int8)
        q[1] = 127
        q[2, 0] = 126
        pad = -k % 16
        store = torch.nn.functional.pad(q, (0, pad)).to(device)
        x = ops.Int8Rows(store[:, :k], torch.ones(3, device=device), dtype=torch.bfloat16)
        y = ops.linear_int8(x, x)
        want = (q.double() @ q.double().t()).float().to(torch.bfloat16)
        assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("device", DEVICES)
def test_linear_int8_rows_with_anything_behind_them(device):
    """Rows cut out of a wider int8 buffer: neither the buffer's other columns nor its rows get in."""
    k, wide = 37, 96
    bx = torch.randint(-127, 128, (9, wide), generator=gen(1), dtype=torch.int8).to(device)
    bw = torch.randint(-127, 128, (21, wide), generator=gen(2), dtype=torch.int8).to(device)
    sx, sw = torch.rand(9, generator=gen(3)).to(device), torch.rand(21, generator=gen(4)).to(device)
    x, w = ops.Int8Rows(bx[:, 16:16 + k], sx, (3, 3, k), torch.float16), ops.Int8Rows(bw[:, 48:48 + k], sw)
    y = ops.linear_int8(x, w)
    assert tuple(y.shape) == (3, 3, 21)
    want, mag = linear64(x.q.cpu(), sx.cpu(), w.q.cpu(), sw.cpu(), None, None, None)
    check(y.reshape(9, 21) * 2.0 ** -8, want * 2.0 ** -8, mag)


@pytest.mark.parametrize("device", DEVICES)
def test_linear_int8_batch_invariance_and_leading_dims(device):
    x = randn(6, 31, 200, seed=7, dtype=torch.bfloat16, device=device)
    w, b = rows(136, 200, 8, device), randn(136, seed=9, dtype=torch.bfloat16, device=device)
    y = ops.linear_int8(x, w, b, act="gelu")
    assert tuple(y.shape) == (6, 31, 136)
    for i in range(6):
        assert torch.equal(ops.linear_int8(x[i], w, b, act="gelu"), y[i])
    assert torch.equal(ops.linear_int8(x[2, 5:6], w, b, act="gelu")[0], y[2, 5])
    assert tuple(ops.linear_int8(x[0, 0], w).shape) == (136,)
    assert tuple(ops.linear_int8(x[:0], w).shape) == (0, 31, 136)


@pytest.mark.parametrize("device", DEVICES)
def test_ln_linear_int8_is_its_two_halves(device):
    x = randn(50, 320, seed=1, dtype=torch.bfloat16, device=device)
    gamma = (1 + 0.1 * randn(320, seed=2)).to(torch.bfloat16).to(device)
    beta = (0.1 * randn(320, seed=3)).to(torch.bfloat16).to(device)
    w = rows(192, 320, 4, device)
    y = ops.ln_linear_int8(x, gamma, beta, 1e-5, w, act="geglu")
    assert torch.equal(y, ops.linear_int8(ops.ln_quantize_rows(x, gamma, beta, 1e-5), w, act="geglu"))


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    bf = torch.bfloat16
    x, w = torch.ones(4, 32, dtype=bf, device=device), rows(8, 32, 1, device)
    i8, one = torch.zeros(4, 32, dtype=torch.int8, device=device), torch.ones(4, device=device)
    for bad in (lambda: ops.Int8Rows(i8.float(), one), lambda: ops.Int8Rows(i8, one.double()),
                lambda: ops.linear_int8(x, x), lambda: ops.linear_int8([1.0], w),
                lambda: ops.quantize_rows(i8)):
        with pytest.raises(TypeError):
            bad()
    odd = torch.zeros(4, 40, dtype=torch.int8, device=device)
    for bad in (lambda: ops.Int8Rows(i8, one[:3]), lambda: ops.Int8Rows(i8[0], one),
                lambda: ops.Int8Rows(odd[:, :32], one), lambda: ops.Int8Rows(i8[:, 1:17], one),
                lambda: ops.Int8Rows(i8.t(), torch.ones(32, device=device)),
                lambda: ops.Int8Rows(i8, one, (4, 31)), lambda: ops.Int8Rows(i8[:, :0], one),
                lambda: ops.Int8Rows(torch.zeros(3 * 32 + 17, dtype=torch.int8, device=device).as_strided(
                    (4, 17), (32, 1)), one),
                lambda: ops.linear_int8(x[:, :16], w), lambda: ops.linear_int8(x, w, act="relu"),
                lambda: ops.linear_int8(x, w, torch.ones(7, dtype=bf, device=device)),
                lambda: ops.linear_int8(x, w, torch.ones(8, device=device)),
                lambda: ops.linear_int8(x, w, residual=torch.ones(4, 7, dtype=bf, device=device)),
                lambda: ops.linear_int8(x, w, residual=torch.ones(4, 8, dtype=bf, device=device), act="geglu"),
                lambda: ops.linear_int8(x, rows(7, 32, 1, device), act="geglu"),
                lambda: ops.quantize_rows(x[:1, :1].expand(2 ** 31, 1)),
                lambda: ops.linear_int8(x[:1].expand(2 ** 31, 32), w),
                lambda: ops.quantize_rows(x[:, :0]), lambda: ops.quantize_rows(torch.ones((), device=device)),
                lambda: ops.quantize_rows(torch.ones(1, ops.INT8_MAX_K + 1, dtype=bf, device=device)),
                lambda: ops.ln_quantize_rows(x, x[0, :16], x[0], 1e-5),
                lambda: ops.ln_quantize_rows(x, x[0].float(), x[0], 1e-5)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="inference only"):
        ops.quantize_rows(torch.ones(2, 32, dtype=bf, device=device, requires_grad=True))
    with pytest.raises(RuntimeError, match="inference only"):
        ops.linear_int8(x, w, torch.ones(8, dtype=bf, device=device, requires_grad=True))


# The kernel of a size follows from its tiles: 256 x 256 from 256 tiles of that kind on, below that two stages from 512
# tiles of 64 x 128 on, four stages under it, all above 16 tokens; rows longer than 640 never take the short-row kernel.
LARGE = {"256 x 256": (4100, 1101, 4099, 4098), "two stages": (2100, 1500, 2050, 2054),
         "four stages": (517, 1101, 1030, 1030)}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,bias,residual", [(None, True, "odd"), (None, False, None), ("gelu", True, "aligned"),
                                               ("quick_gelu", False, "odd"), ("geglu", True, None)])
@pytest.mark.parametrize("name", LARGE)
def test_every_kernel_of_large_products(cuda, dtype, act, bias, residual, name):
    """Widths that are no multiple of a vector, rows that are none of 16 bytes, residuals at odd elements: the
    element-wise epilogue of every tile kernel; the same with a width of whole vectors."""
    dt, (m, k, odd, glu) = DTYPES[dtype], LARGE[name]
    tiles = lambda bm, bn, n: -(-m // bm) * -(-n // bn)     # noqa: E731
    for n in ((glu if act == "geglu" else odd), (glu if act == "geglu" else odd) // 16 * 16):
        want_kernel = ("256 x 256" if tiles(256, 256, n) >= 256 else
                       "two stages" if tiles(64, 128, n) >= 512 else "four stages")
        assert want_kernel == name and m > 16 and k > 640
        x, w = randn(m, k, seed=1, dtype=dt, device=cuda) * 2, rows(n, k, 2, cuda, dt)
        b = randn(n, seed=3, dtype=dt, device=cuda) if bias else None
        store = randn(m * n + 8, seed=4, dtype=dt, device=cuda) if residual else None
        r = None if store is None else store[(1 if residual == "odd" else 8):][:m * n].view(m, n)
        q = ops.quantize_rows(x)
        y = ops.linear_int8(x, w, b, residual=r, act=act)
        want, mag = linear64(q.q, q.scale, w.q, w.scale, b, r, act)
        over = (y.double() - want).abs() - (torch.finfo(dt).eps / 2 * want.abs() + 2.0 ** -20 * mag + 2.0 ** -25)
        assert bool((over <= 0).all()), f"n {n}: over the bound by {over.max().item():.3g}"
        assert torch.equal(ops.linear_int8(q, w, b, residual=r, act=act), y)


@pytest.mark.gpu
def test_gpu_types_refused(cuda):
    with pytest.raises(TypeError):
        ops.quantize_rows(torch.ones(2, 32, device=cuda))
    w = rows(8, 32, 1, cuda)
    with pytest.raises(TypeError):
        ops.linear_int8(ops.Int8Rows(w.q, w.scale, dtype=torch.float32), w)
    with pytest.raises(ValueError):
        ops.linear_int8(torch.ones(2, 32, dtype=torch.bfloat16), w)


# ------------------------------------------------------------------ as a model uses it
class _Block(nn.Module):
    def __init__(self):
        super().__init__()
        self.ln, self.fc1, self.fc2 = layers.LayerNorm(96), layers.Linear(96, 200), layers.Linear(200, 96)

    def forward(self, x):
        return self.fc2(self.ln.linear(x, self.fc1, act="gelu"), residual=x)


@pytest.mark.parametrize("device", DEVICES)
def test_layers_in_8_bits(device):
    m = layers.init_weights(_Block(), 3).to(device=device, dtype=torch.bfloat16)
    x = randn(2, 11, 96, seed=6, dtype=torch.bfloat16, device=device)
    before = m(x)
    assert layers.int8_linears(m) == 2
    y = m(x)
    h = ops.ln_linear_int8(x, m.ln.weight, m.ln.bias, m.ln.eps, ops.quantize_rows(m.fc1.weight), m.fc1.bias,
                           act="gelu")
    assert torch.equal(y, ops.linear_int8(h, ops.quantize_rows(m.fc2.weight), m.fc2.bias, residual=x))
    # 8-bit weights and activations: each operand is off by at most half of 1/127 of its row's largest value
    assert (y.float() - before.float()).norm() < 0.03 * before.float().norm()
    layers.int8_linears(m, False)
    assert torch.equal(m(x), before)


@pytest.mark.parametrize("device", DEVICES)
def test_layers_in_8_bits_are_published_when_they_are_ready(device, monkeypatch):
    """Forks on other streams share the layers: none is switched before the kernels of all have finished, and none
    where a later one cannot be."""
    m = layers.init_weights(_Block(), 3).to(device=device, dtype=torch.bfloat16)
    seen = []

    def ready(t):
        seen.append((t.device, [lin.int8 for lin in (m.fc1, m.fc2)]))
    monkeypatch.setattr(ops, "derived_ready", ready)
    layers.int8_linears(m)
    assert seen == [(m.fc1.weight.device, [None, None])] and m.fc1.int8 is not None and m.fc2.int8 is not None
    layers.int8_linears(m, False)
    m.fc2.weight = nn.Parameter(m.fc2.weight.int(), requires_grad=False)
    with pytest.raises(TypeError):
        layers.int8_linears(m)
    assert m.fc1.int8 is None


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("b,n,c", [(2, 64, 64), (1, 4096, 320)])
def test_layers_behind_a_group_norm_in_8_bits(device, b, n, c):
    """GroupNorm then linear, a GEGLU projection without a norm: 8 bits where the layer is switched."""
    lin = layers.init_weights(nn.ModuleList([layers.Linear(c, 96)]), 3)[0].to(device=device, dtype=torch.bfloat16)
    norm = layers.init_weights(nn.ModuleList([layers.GroupNorm(8, c)]), 4)[0].to(device=device, dtype=torch.bfloat16)
    x = (randn(b, n, c, seed=6, device=device) * 2 + 1).to(torch.bfloat16)
    want, gate = lin.forward_norm(x, norm.table(x, silu=True)), lin.geglu(x)
    assert layers.int8_linears(lin) == 1
    got = lin.forward_norm(x, norm.table(x, silu=True))
    assert torch.equal(got, ops.linear_int8(ops.normed(x, norm.table(x, silu=True)), lin.int8, lin.bias))
    # both operands off by at most half of 1/127 of their row's largest value
    assert 0 < (got.float() - want.float()).norm() < 0.03 * want.float().norm()
    assert torch.equal(lin.geglu(x), ops.linear_int8(x, lin.int8, lin.bias, act="geglu"))
    assert 0 < (lin.geglu(x).float() - gate.float()).norm() < 2 * 0.03 * gate.float().norm()     # a product of two


def test_layers_counted_are_those_that_run_in_8_bits():
    """Every layer that int8_linears counts runs in 8 bits in a forward pass of the UNet; the time projections, batched
    through their bare weights, are not among them."""
    from arbius_amd.models.unet2d import ResBlock, UNet2DCondition, UNetConfig
    unet = layers.init_weights(UNet2DCondition(UNetConfig.tiny()), 1).eval()
    count = layers.int8_linears(unet)
    with layers.Int8Uses() as uses:
        unet(randn(1, 8, 8, 4, seed=1), torch.tensor([5.0]), randn(1, 7, 32, seed=2))
    assert count == len(uses.forms) and all(form is not None for _, form in uses.forms.values())
    assert all(m.temb_proj.int8 is None for m in unet.modules() if isinstance(m, ResBlock))


@pytest.mark.parametrize("device", DEVICES)
def test_weights_that_change_are_quantised_again(device):
    """Loaded, changed in place, cast: no layer answers with the 8-bit form of values it no longer has."""
    m, other = (layers.init_weights(_Block(), s).to(device=device, dtype=torch.bfloat16) for s in (3, 4))
    x = randn(5, 96, seed=6, dtype=torch.bfloat16, device=device)

    def fresh():
        again = layers.init_weights(_Block(), 0).to(device=device, dtype=m.fc1.weight.dtype)
        again.load_state_dict(m.state_dict())
        layers.int8_linears(again)
        return again
    layers.int8_linears(m)
    first = m(x)
    m.load_state_dict(other.state_dict())
    assert torch.equal(m(x), fresh()(x)) and not torch.equal(m(x), first)
    with torch.no_grad():
        m.fc2.weight.mul_(2.0)
    assert torch.equal(m(x), fresh()(x))
    m.to(torch.float16)
    assert torch.equal(m(x.half()), fresh()(x.half()))
    held = m.fc1.int8
    m(x.half())
    assert m.fc1.int8 is held


def test_a_capture_knows_the_forms_it_used():
    """What a captured graph keeps of the layers it ran: the 8-bit weights themselves, and whether they still are the
    layers' weights."""
    m, other = (layers.init_weights(_Block(), s) for s in (3, 4))
    x = randn(3, 96, seed=6)

    def capture():
        with layers.Int8Uses() as uses:
            m(x)
        return uses
    a = capture()
    assert set(a.forms.values()) == {(m.fc1, None), (m.fc2, None)} and a.current()
    layers.int8_linears(other)                               # not its layers
    assert a.current()
    layers.int8_linears(m.fc2)
    assert not a.current()
    b = capture()
    assert b.current() and (m.fc2, m.fc2.int8) in b.forms.values()
    layers.int8_linears(m.fc2)                               # quantised again: other tensors
    assert not b.current() and not a.current()
    m.fc2.int8 = None
    assert a.current() and not b.current()
    layers.int8_linears(m)
    c = capture()
    assert c.current()
    m.load_state_dict(other.state_dict())                    # other weights
    assert not c.current()
    d = capture()
    assert d.current() and not c.current()
    layers.int8_linears(m, False)
    m(x)                                                     # outside of a capture nothing is noted
    assert len(a.forms) == 2


@pytest.mark.gpu
def test_captured_graphs_follow_the_layers(cuda):
    """Switched on, quantised again after a weight change and off: pipelines and their forks, with graphs captured
    before, answer as the eager model does, whatever was allocated where the old 8-bit weights were."""
    from arbius_amd.models.registry import build_pipeline
    pipe = build_pipeline("anythingv3", device=cuda, use_graphs=True)
    fork, eager = pipe.fork(), pipe.fork()
    eager.use_graphs = False
    eager._reset_graphs()
    kw = dict(prompt="a lake", width=128, height=128, num_inference_steps=2, scheduler="DPMSolverMultistep", seed=7)
    images, kept = [], []

    def solve():
        want = eager(**kw)
        kept.append([torch.full((1 << 20,), 85, dtype=torch.uint8, device=cuda) for _ in range(64)])
        for p in (pipe, fork, pipe):
            assert (p(**kw) == want).all()
        images.append(want)
    solve()
    assert sum(layers.int8_linears(m) for m in (pipe.unet, pipe.text)) > 150
    solve()
    with torch.no_grad():
        for layer in pipe.text.layers:
            layer.fc2.weight.mul_(0.5)
    layers.int8_linears(pipe.text)
    solve()
    for m in (pipe.unet, pipe.text):
        layers.int8_linears(m, False)
    solve()
    assert all((a != b).any() for i, a in enumerate(images) for b in images[:i])


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_forks_in_8_bits_at_once(cuda, graphs):
    """Two forks on their own threads and streams whose first use of changed weights comes at once: what each answers
    alone afterwards."""
    from concurrent.futures import ThreadPoolExecutor
    from arbius_amd.models.registry import build_pipeline
    pipe = build_pipeline("anythingv3", device=cuda, use_graphs=graphs)
    for m in (pipe.unet, pipe.text):
        layers.int8_linears(m)
    kws = [dict(prompt=f"a lake {i}", width=128, height=128, num_inference_steps=2, scheduler="DPMSolverMultistep",
                seed=i) for i in range(2)]
    forks, last = [pipe.fork() for _ in kws], None
    for _ in range(3):
        with torch.no_grad():
            for m in (*pipe.text.modules(), *pipe.unet.modules()):
                if isinstance(m, layers.Linear):
                    m.weight.mul_(1.0625)
        torch.cuda.synchronize()
        with ThreadPoolExecutor(2) as ex:
            got = list(ex.map(lambda a: a[0](**a[1]), zip(forks, kws)))
        want = [pipe(**kw) for kw in kws]
        assert all((g == w).all() for g, w in zip(got, want))
        assert last is None or (last != want[0]).any()
        last = want[0]


@pytest.mark.gpu
def test_a_graph_of_other_forms_is_refused(cuda):
    from arbius_amd.models.graphs import GraphCache, GraphedCall
    m = layers.init_weights(_Block(), 3).to(device=cuda, dtype=torch.bfloat16)
    x = randn(5, 96, seed=6, dtype=torch.bfloat16, device=cuda)
    cache, want = GraphCache(m, True), m(x)
    old = GraphedCall(m, [x])
    assert torch.equal(cache(x), want) and torch.equal(old(x), want)
    layers.int8_linears(m)
    with pytest.raises(RuntimeError, match="8 bits"):
        old(x)
    want8 = m(x)
    assert torch.equal(cache(x), want8) and not torch.equal(want, want8)
    layers.int8_linears(m, False)
    assert torch.equal(cache(x), want) and torch.equal(old(x), want)
    layers.int8_linears(m)
    old = GraphedCall(m, [x])
    assert torch.equal(cache(x), want8) and torch.equal(old(x), want8)
    m.load_state_dict(layers.init_weights(_Block(), 5).state_dict())
    with pytest.raises(RuntimeError, match="8 bits"):
        old(x)
    got = cache(x).clone()
    assert torch.equal(got, m(x)) and not torch.equal(got, want8)


@pytest.mark.gpu
def test_streams_and_graph_replays(cuda):
    x = randn(33, 640, seed=1, dtype=torch.bfloat16, device=cuda)
    w, b = rows(384, 640, 2, cuda), randn(384, seed=3, dtype=torch.bfloat16, device=cuda)
    want = ops.linear_int8(x, w, b, act="geglu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.linear_int8(x, w, b, act="geglu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    xs, graphs = [x.clone(), x.clone()], []
    for i in range(2):                    # two graphs of the same weight, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.linear_int8(xs[i], w, b, act="geglu")
        graphs.append((g, y))
    for step in range(4):
        for i in range(2):
            xs[i].copy_(randn(33, 640, seed=10 * step + i, dtype=torch.bfloat16, device=cuda))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(graphs[i][1], ops.linear_int8(xs[i], w, b, act="geglu"))


@pytest.mark.gpu
def test_more_rows_than_a_grid_dimension(cuda):
    m = 70001
    x = randn(64, 48, seed=1, dtype=torch.bfloat16, device=cuda).repeat(-(-m // 64), 1)[:m]
    w = rows(40, 48, 2, cuda)
    y = ops.linear_int8(x, w)
    assert torch.equal(y[:64].repeat(-(-m // 64), 1)[:m], y)


# ------------------------------------------------------------------ few tokens
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [None, "geglu"])
@pytest.mark.parametrize("k,n", [(8, 2), (72, 34), (640, 520), (2048, 96), (8184, 66), (8192, 40), (8200, 40),
                                 (77, 30)])
def test_few_tokens(device, dtype, act, k, n):
    """1 to 17 tokens around every switch of kernels: rows quantised inside the product or apart give the same bits,
    also zero rows, rows with NaN or infinity, and rows cut out of wider ones."""
    dt = DTYPES[dtype]
    wide = randn(17, k + 24, seed=k, dtype=dt, device=device)
    wide[2], wide[3, 9] = 0, float("nan")
    if k > 8:
        wide[1, -25], wide[5, 8] = float("inf"), -float("inf")
    w, b = rows(n, k, n, device, dt), randn(n, seed=1, dtype=dt, device=device)
    for m in (1, 2, 3, 4, 5, 17):
        for x in (wide[:m, 8:8 + k], wide[:m, 3:3 + k], wide[17 - m:, 8:8 + k].clone(), wide[2:3, 8:8 + k]):
            qx = ops.quantize_rows(x)
            y = ops.linear_int8(x, w, b, act=act)
            assert torch.equal(y.nan_to_num(7.0), ops.linear_int8(qx, w, b, act=act).nan_to_num(7.0))
            fine = qx.scale.isfinite().cpu()
            assert torch.equal(y.cpu().isnan().any(dim=1), ~fine)
            check(y.cpu()[fine], *linear64(qx.q.cpu()[fine], qx.scale.cpu()[fine], w.q.cpu(), w.scale.cpu(), b.cpu(),
                                           None, act))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("k", [320, 2048, 1001])
def test_layernorm_batch_invariance(device, k):
    x = randn(300, k, seed=1, dtype=torch.bfloat16, device=device)
    gamma, beta = (1 + 0.1 * randn(k, seed=2)).to(x), (0.1 * randn(k, seed=3)).to(x)
    w = rows(72, k, 4, device)
    y, q = ops.ln_linear_int8(x, gamma, beta, 1e-5, w), ops.ln_quantize_rows(x, gamma, beta, 1e-5)
    for a, e in ((0, 1), (7, 8), (20, 24), (3, 70), (100, 300)):
        assert torch.equal(ops.ln_linear_int8(x[a:e], gamma, beta, 1e-5, w), y[a:e])
        part = ops.ln_quantize_rows(x[a:e], gamma, beta, 1e-5)
        assert torch.equal(part.q, q.q[a:e]) and torch.equal(part.scale, q.scale[a:e])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [8, 312, 320, 328, 640, 1000, 1280, 2048, 2560, 4096, 8192, 16384, 16392, 1001])
def test_layernorm_order_is_the_lengths_alone(device, dtype, k):
    """The same rows at an odd base, with a row stride that is no multiple of a vector, or alone, behind gamma and
    beta at odd bases: the same 8 bits, scales and products."""
    dt, m = DTYPES[dtype], 200 if k < 4000 else 40
    x = (randn(m, k, seed=1) * 3 + 0.5).to(dt).to(device)
    gamma, beta = (1 + 0.1 * randn(k, seed=2)).to(dt).to(device), (0.1 * randn(k, seed=3)).to(dt).to(device)
    w = rows(40, k, 4, device, dt)
    odd, apart = torch.empty(m * k + 1, dtype=dt, device=device)[1:].view(m, k), \
        torch.empty(m, k + 5, dtype=dt, device=device)[:, :k]
    odd.copy_(x)
    apart.copy_(x)
    go, bo = (torch.cat([t[:1], t])[1:] for t in (gamma, beta))
    want, y = ops.ln_quantize_rows(x, gamma, beta, 1e-5), ops.ln_linear_int8(x, gamma, beta, 1e-5, w)
    for xs, g, b in ((odd, gamma, beta), (apart, gamma, beta), (x, go, beta), (x, gamma, bo), (apart, go, bo)):
        got = ops.ln_quantize_rows(xs, g, b, 1e-5)
        assert torch.equal(got.scale, want.scale) and torch.equal(got.q, want.q)
        assert torch.equal(ops.ln_linear_int8(xs, g, b, 1e-5, w), y)
        for i in (0, 7, m - 1):
            one = ops.ln_quantize_rows(xs[i], g, b, 1e-5)
            assert torch.equal(one.scale, want.scale[i:i + 1]) and torch.equal(one.q[0], want.q[i])


@pytest.mark.gpu
@pytest.mark.parametrize("k", [320, 640])
def test_many_short_rows_behind_a_layernorm_at_any_address(cuda, k):
    """The kernel of many short rows takes aligned rows only; what it refuses gives the same bits."""
    m, bf = 33000, torch.bfloat16
    x = randn(m, k, seed=1, dtype=bf, device=cuda)
    gamma, beta = (1 + 0.1 * randn(k, seed=2)).to(x), (0.1 * randn(k, seed=3)).to(x)
    w = rows(136, k, 4, cuda)
    apart = torch.empty(m, k + 4, dtype=bf, device=cuda)[:, :k]
    apart.copy_(x)
    y = ops.ln_linear_int8(x, gamma, beta, 1e-5, w)
    assert torch.equal(ops.ln_linear_int8(apart, gamma, beta, 1e-5, w), y)
    assert torch.equal(ops.ln_linear_int8(apart[5], gamma, beta, 1e-5, w), y[5])


@pytest.mark.parametrize("device", DEVICES)
def test_operands_of_any_alignment(device):
    """Bias and residual cut out of others at odd elements, results whose width is no multiple of a vector."""
    for m, k, n in ((3, 64, 70), (70, 200, 136), (300, 128, 520)):
        x, w = randn(m, k, seed=1, dtype=torch.bfloat16, device=device), rows(n, k, 2, device)
        b = randn(n + 1, seed=3, dtype=torch.bfloat16, device=device)[1:]
        store = randn(m * n + 3, seed=4, dtype=torch.bfloat16, device=device)
        for r in (store[3:].view(m, n), store[1:1 + m * n].view(n, m).t(), store[:n].expand(m, n)):
            y = ops.linear_int8(x, w, b, residual=r)
            assert torch.equal(y, ops.linear_int8(x, w, b.clone(), residual=r.contiguous()))


@pytest.mark.gpu
def test_few_tokens_in_a_graph(cuda):
    x, w = randn(2, 640, seed=1, dtype=torch.float16, device=cuda), rows(384, 640, 2, cuda, torch.float16)
    ops.linear_int8(x, w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.linear_int8(x, w)
    for step in range(4):
        x.copy_(randn(2, 640, seed=5 + step, dtype=torch.float16))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.linear_int8(ops.quantize_rows(x), w))


# ------------------------------------------------------------------ many short rows
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ln", [False, True])
@pytest.mark.parametrize("act", [None, "gelu", "quick_gelu", "geglu"])
@pytest.mark.parametrize("m,k,n", [(8192, 320, 192), (32769, 312, 80), (32800, 64, 1040), (32900, 8, 16),
                                   (33221, 640, 400), (32768, 328, 48), (32768, 576, 2064), (40000, 160, 32),
                                   (32790, 320, 1984)])
def test_many_short_rows(device, dtype, ln, act, m, k, n):
    """Rows quantised (and normalised) inside the product: bit for bit the two operators apart, with zero rows, rows
    with NaN or infinity, rows cut out of wider ones."""
    dt = DTYPES[dtype]
    if device == "cpu":
        m = m % 100 + 8
    x = randn(64, k + 8, seed=k, dtype=dt, device=device).repeat(-(-m // 64), 1)[:m, 8:]
    x[:, ::5] *= torch.linspace(0.1, 3, m, device=device)[:, None].to(dt)
    x[3], x[m - 2], x[5, k - 1], x[m - 1, 0] = 0, 0, float("nan"), float("inf")
    gamma, beta = (1 + 0.1 * randn(k, seed=2)).to(x), (0.1 * randn(k, seed=3)).to(x)
    w, b = rows(n, k, 4, device, dt), randn(n, seed=5, dtype=dt, device=device)
    res = randn(m, n, seed=6, dtype=dt, device=device)
    for bias, r in ((b, None), (None, None if act == "geglu" else res)):
        if ln:
            y = ops.ln_linear_int8(x, gamma, beta, 1e-5, w, bias, residual=r, act=act)
            q = ops.ln_quantize_rows(x, gamma, beta, 1e-5)
        else:
            y, q = ops.linear_int8(x, w, bias, residual=r, act=act), ops.quantize_rows(x)
        want = ops.linear_int8(q, w, bias, residual=r, act=act)
        bad = torch.zeros(m, dtype=torch.bool, device=device)
        bad[5] = bad[m - 1] = True
        assert torch.equal(y.isnan().all(dim=1), bad) and torch.equal(y[~bad], want[~bad])


@pytest.mark.gpu
def test_many_short_rows_in_a_graph(cuda):
    x, w = randn(32800, 320, seed=1, dtype=torch.bfloat16, device=cuda), rows(384, 320, 2, cuda)
    gamma, beta = torch.ones(320, device=cuda).to(x), torch.zeros(320, device=cuda).to(x)
    ops.ln_linear_int8(x, gamma, beta, 1e-5, w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.ln_linear_int8(x, gamma, beta, 1e-5, w)
        z = ops.linear_int8(x, w, act="geglu")
    for step in range(4):
        x.copy_(randn(32800, 320, seed=5 + step, dtype=torch.bfloat16))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.linear_int8(ops.ln_quantize_rows(x, gamma, beta, 1e-5), w))
        assert torch.equal(z, ops.linear_int8(ops.quantize_rows(x), w, act="geglu"))
