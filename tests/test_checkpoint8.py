"""8-bit activation checkpoints (ops.checkpoint8) against their definition in 64 bits.

Codes and values are exact: they are compared bit for bit. Products: an output
of type t is off by its rounding, eps(t)/2 of the value, and a 32-bit sum of n
products by at most n 2^-23 times the sum of their magnitudes.
"""
import pytest
import torch

from gordo_amd.ops import Saved8, gated_scan, linear8, load8, save8, weight_grad8

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


def kept8(v):
    """[..., F] as float64, as 8-bit codes keep it."""
    v = v.detach().cpu().double()
    out = torch.empty_like(v)
    for at in range(0, v.shape[-1], 32):
        w = v[..., at : at + 32]
        _, e = torch.frexp(w.abs().amax(-1, keepdim=True))
        step = torch.exp2((e - 7).clamp_min(-126).double())
        q = torch.clamp(torch.round(w / step), -127, 127) * step
        out[..., at : at + 32] = torch.where(torch.isfinite(w).all(-1, keepdim=True), q, float("nan"))
    return out


def values(N, F, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, F, generator=g) * torch.exp(2 * torch.randn(N, F, generator=g))
    return x.to(dtype).to(device)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0)) and torch.equal(a.isnan(), b.isnan())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N,F", [(1, 1), (1, 31), (3, 32), (2, 33), (5, 50), (7, 64), (257, 96), (130, 1000), (4, 2050)])
def test_round_trip(device, dtype, N, F):
    x = values(N, F, dtype, device)
    saved = save8(x)
    assert saved.codes.shape == (N, -(-F // 32) * 32) and saved.scales.shape == (N, -(-F // 32))
    got = load8(saved)
    assert got.dtype == dtype and torch.equal(got.cpu().double(), kept8(x))
    assert saved.codes.abs().max() <= 127 and not saved.codes[:, F:].any()
    group = torch.nn.functional.pad(x.cpu().double(), (0, -F % 32)).reshape(N, -1, 32)
    off = torch.nn.functional.pad((got - x).cpu().double(), (0, -F % 32)).reshape(N, -1, 32)
    assert (off.abs().amax(-1) <= group.abs().amax(-1) / 127 + 2.0**-127).all()
    for wide in (torch.float32, torch.bfloat16):
        assert torch.equal(load8(saved, wide).double(), got.double())  # exact in both
    assert torch.equal(load8(save8(got)), got)  # what was kept once is kept as it is


@pytest.mark.parametrize("device", DEVICES)
def test_edges_of_the_range(device):
    """Zeros, subnormal numbers, the largest ones, and borders between two codes and two scales."""
    tiny, top = 2.0**-149, torch.finfo(torch.float32).max
    rows = [
        [0.0, -0.0] * 16,
        [tiny, -3 * tiny] * 16,
        [2.0**-126, 2.0**-127, 2.0**-120, 2.0**-121] * 8,
        [top, -top, 1.0, top / 127] * 8,
        [63.5, 64.5, 0.5, 1.5, 126.5, 127.49, 127.51, -127.99] * 4,
        [1.0] + [2.0**-7, 3 * 2.0**-7, 2.0**-8] * 10 + [0.0],
        [1.0 - 2.0**-24, 0.5, -0.25, 0.126] * 8,
    ]
    x = torch.tensor(rows, device=device)
    got = load8(save8(x))
    assert torch.equal(got.cpu().double(), kept8(x)) and torch.isfinite(got).all()
    h = torch.tensor([[65504.0, -65504.0, 6e-8, 512.0] * 8, [2.0**-24, 2.0**-23, -(2.0**-24), 0.0] * 8], dtype=torch.float16, device=device)
    got = load8(save8(h))
    assert torch.equal(got.cpu().double(), kept8(h)) and torch.isfinite(got).all()
    assert torch.equal(got[1], h[1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_not_finite_stays_in_its_group(device, dtype, bad):
    x = values(4, 80, dtype, device)
    x[1, 40], x[3, 79] = bad, bad
    got = load8(save8(x))
    assert same(got.cpu().double(), kept8(x))
    assert got[1, 32:64].isnan().all() and got[3, 64:].isnan().all() and int(got.isnan().sum()) == 48


@pytest.mark.parametrize("device", DEVICES)
def test_shapes_and_strides(device):
    x = values(24, 40, torch.bfloat16, device)
    want = load8(save8(x))
    three = x.reshape(2, 12, 40)
    assert torch.equal(load8(save8(three)), want.reshape(2, 12, 40))
    assert torch.equal(load8(save8(three.transpose(0, 1))), want.reshape(2, 12, 40).transpose(0, 1))
    wide = torch.full((24, 47), 1e6, dtype=x.dtype, device=device)
    wide[:, 3:43] = x
    assert torch.equal(load8(save8(wide[:, 3:43])), want)
    assert torch.equal(load8(save8(x.t().contiguous().t())), want)
    assert torch.equal(load8(save8(x[::2])), want[::2])
    assert load8(save8(x[:0])).shape == (0, 40)
    assert torch.equal(load8(save8(x[0])), want[0])
    column = x[:, 5:6]
    assert torch.equal(load8(save8(column)).double().cpu(), kept8(column))


def test_checkpoint_refuses():
    x = torch.randn(4, 40)
    s = save8(x)
    for bad in (
        lambda: save8(x.double()),
        lambda: save8(x.to(torch.int8)),
        lambda: save8(torch.tensor(1.0)),
        lambda: save8(x[:, :0]),
        lambda: save8([1.0]),
        lambda: load8(x),
        lambda: load8(s, torch.float64),
        lambda: load8(Saved8(s.codes, s.scales, torch.Size([4, 70]), s.dtype)),
        lambda: load8(Saved8(s.codes[:3], s.scales, s.shape, s.dtype)),
        lambda: load8(Saved8(s.codes.float(), s.scales, s.shape, s.dtype)),
        lambda: load8(Saved8(s.codes, s.scales, torch.Size([4, 0]), s.dtype)),
        lambda: load8(Saved8(s.codes, s.scales, torch.Size([]), s.dtype)),
        lambda: load8(Saved8(s.codes, s.scales, s.shape, torch.int8), torch.float32),
        lambda: weight_grad8(torch.randn(5, 3), s),
        lambda: weight_grad8(torch.randn(2, 2, 3), s),
        lambda: weight_grad8(torch.randn(4, 3).double(), s),
        lambda: weight_grad8(torch.randn(4, 3), s, dtype=torch.int32),
        lambda: weight_grad8(torch.randn(4, 3, device="meta"), s),
        lambda: linear8(x, torch.randn(3, 41)),
        lambda: linear8(x, torch.randn(3, 40), torch.randn(4)),
        lambda: linear8(x, torch.randn(40)),
        lambda: linear8(x, torch.randn(0, 40)),
        lambda: linear8(x.double(), torch.randn(3, 40).double()),
        lambda: linear8(x, torch.randn(3, 40, device="meta")),
    ):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------- linear layer
def close(got, want, magnitude, n, what, steps=0.5):
    """`magnitude`: sum of the magnitudes of what was summed, for each output;
    `steps`: roundings to got's type on the way, in its half steps."""
    got = got.detach().cpu()
    assert got.shape == want.shape, what
    eps = torch.finfo(got.dtype).eps
    allowed = steps * eps * want.abs() * 1.01 + n * 2.0**-23 * magnitude + 1e-37
    if got.dtype == torch.float16:
        allowed = allowed + 2.0**-25
    off = (got.double() - want).abs() - allowed
    assert not off.numel() or float(off.max()) <= 0, (what, float(off.max()))


def check_weight_grad(dy, x, dtype, bias=True):
    dw, db = weight_grad8(dy, save8(x), bias=bias, dtype=dtype)
    d, q = dy.detach().cpu().double().reshape(-1, dy.shape[-1]), kept8(x).reshape(-1, x.shape[-1])
    n = len(d)
    close(dw, d.t() @ q, d.abs().t() @ q.abs(), n, "dw")
    if bias:
        close(db, d.sum(0), d.abs().sum(0), n, "db")
    else:
        assert db is None
    return dw, db


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize(
    "N,F,O", [(1, 1, 1), (3, 5, 2), (31, 33, 17), (64, 64, 64), (65, 50, 38), (257, 130, 129), (100, 256, 16), (1030, 40, 300), (2049, 127, 65)]
)
def test_weight_gradient(device, dtype, N, F, O):
    g = torch.Generator().manual_seed(N)
    dy = torch.randn(N, O, generator=g).to(dtype).to(device)
    check_weight_grad(dy, values(N, F, dtype, device).clamp(-100, 100), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("N,F,O", [(12000, 300, 520), (12001, 301, 517), (11000, 512, 512), (600, 1500, 2100)])
def test_weight_gradient_of_wide_layers(dtype, N, F, O):
    g = torch.Generator().manual_seed(N)
    dy = torch.randn(N, O, generator=g).to(dtype).cuda()
    check_weight_grad(dy, torch.randn(N, F, generator=g).to(dtype).cuda(), dtype)
    check_weight_grad(dy, torch.randn(N, F, generator=g).to(dtype).cuda(), torch.float32, bias=False)


@pytest.mark.parametrize("device", DEVICES)
def test_weight_gradient_of_values_beyond_float16(device):
    """dy in float16 beside an input that was kept from float32."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(50, 40, generator=g).to(device) * 2.0**40
    dy = torch.randn(50, 24, generator=g).to(torch.float16).to(device)
    check_weight_grad(dy, x, torch.float32)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_weight_gradient_of_the_largest_values(device, dtype):
    """Inputs up to the largest finite number, whose steps are 2^121."""
    g = torch.Generator().manual_seed(8)
    x = (torch.rand(70, 40, generator=g) * 2 - 1) * torch.finfo(dtype).max
    dy = torch.randn(70, 33, generator=g) * 2.0**-100
    dw, _ = check_weight_grad(dy.to(dtype).to(device), x.to(dtype).to(device), torch.float32)
    assert dw.isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
def test_the_largest_32_bit_gradient(device):
    """A finite gradient stays finite where the next bf16 number is infinite."""
    top = torch.finfo(torch.float32).max
    g = torch.Generator().manual_seed(9)
    dy = torch.stack([torch.full((5,), top), torch.full((5,), -top)]).to(device)
    x = (torch.randn(2, 40, generator=g) * 2.0**-100).to(device)
    dw, db = check_weight_grad(dy, x, torch.float32)
    assert dw.isfinite().all() and not db.any()
    check_weight_grad(dy[:1], x[:1], torch.float32)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("of_dy", DTYPES, ids=str)
@pytest.mark.parametrize("to", DTYPES, ids=str)
@pytest.mark.parametrize("N", [70, 3001])
def test_weight_gradient_types(device, of_dy, to, N):
    """Every type of dy to every type of gradient, whole and in parts that are joined."""
    g = torch.Generator().manual_seed(1)
    dy = torch.randn(N, 48, generator=g).to(of_dy).to(device)
    x = torch.randn(N, 72, generator=g).to(of_dy).to(device)
    check_weight_grad(dy, x, to)
    check_weight_grad(dy, x, to, bias=False)


@pytest.mark.parametrize("device", DEVICES)
def test_weight_gradient_strides(device):
    g = torch.Generator().manual_seed(2)
    N, F, O = 90, 40, 24
    x = torch.randn(N, F, generator=g).to(torch.bfloat16).to(device)
    wide = torch.full((N, O + 9), float("nan"), dtype=x.dtype, device=device)
    for first in (0, 1, 4, 8):
        dy = wide[:, first : first + O]
        dy.copy_(torch.randn(N, O, generator=g))
        check_weight_grad(dy, x, x.dtype)
        wide.fill_(float("nan"))
    dy = torch.randn(O, N, generator=g).to(x.dtype).to(device).t()
    check_weight_grad(dy, x, x.dtype)
    check_weight_grad(torch.ones(1, O, dtype=x.dtype, device=device).expand(N, O), x, x.dtype)
    three = torch.randn(9, 10, O, generator=g).to(x.dtype).to(device)
    check_weight_grad(three, x.reshape(9, 10, F), x.dtype)


@pytest.mark.parametrize("device", DEVICES)
def test_weight_gradient_of_nothing(device):
    dw, db = weight_grad8(torch.randn(0, 5, device=device), save8(torch.randn(0, 40, device=device)), bias=True)
    assert dw.shape == (5, 40) and not dw.any() and not db.any()


@pytest.mark.parametrize("device", DEVICES)
def test_weight_gradient_carries_nan(device):
    """A group that was not finite reaches its own columns and no others."""
    x = torch.randn(40, 96, device=device)
    x[7, 40] = float("inf")
    dw, _ = weight_grad8(torch.randn(40, 33, device=device), save8(x))
    assert dw[:, 32:64].isnan().all() and torch.isfinite(dw[:, :32]).all() and torch.isfinite(dw[:, 64:]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_32_bit_gradient_keeps_32_bits(device):
    """dy = 1 + 2^-20: half of it lies below what two bf16 numbers hold."""
    dy = torch.full((64, 32), 1 + 2.0**-20, device=device)
    dy[1::2] = -1.0
    x = torch.ones(64, 32, device=device)
    dw, db = weight_grad8(dy, save8(x), bias=True)
    # partial sums are below 64 and multiples of 2^-20: exact in 32 bits... of which 24 hold 2^-18 above 32
    assert (dw.cpu().double() - 32 * 2.0**-20).abs().max() <= 64 * 2.0**-24
    assert (db.cpu().double() - 32 * 2.0**-20).abs().max() <= 64 * 2.0**-24


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("master", [False, True], ids=["one type", "32-bit weights"])
def test_linear8(device, dtype, master):
    g = torch.Generator().manual_seed(5)
    to = torch.float32 if master else dtype
    x = torch.randn(3, 21, 50, generator=g).to(dtype).to(device).requires_grad_()
    w = (torch.randn(38, 50, generator=g) / 7).to(to).to(device).requires_grad_()
    b = torch.randn(38, generator=g).to(to).to(device).requires_grad_()
    dy = torch.randn(3, 21, 38, generator=g).to(dtype).to(device)
    y = linear8(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert (y.dtype, dx.dtype, dw.dtype, db.dtype) == (dtype, dtype, to, to)
    X, W, B_, D = (t.detach().to(dtype).cpu().double() for t in (x, w, b, dy))
    close(y, X @ W.t() + B_, X.abs() @ W.abs().t() + B_.abs(), 51, "y", steps=1.0)
    close(dx, D @ W, D.abs() @ W.abs(), 38, "dx", steps=1.0)
    D2, Q = D.reshape(-1, 38), kept8(x).reshape(-1, 50)
    close(dw, D2.t() @ Q, D2.abs().t() @ Q.abs(), 63, "dw")
    close(db, D2.sum(0), D2.abs().sum(0), 63, "db")


@pytest.mark.parametrize("device", DEVICES)
def test_linear8_parts(device):
    """No bias, frozen weights, a frozen input, and what stays alive for the backward pass."""
    x, w = torch.randn(30, 64, device=device), torch.randn(8, 64, device=device)
    b = torch.randn(8, device=device)
    y = linear8(x, w.clone().requires_grad_())
    assert torch.allclose(y, x @ w.t(), atol=1e-4)
    xr = x.clone().requires_grad_()
    kept = []
    watch = torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t)
    with watch:
        y = linear8(xr, w, b)
    assert [t.shape for t in kept] == [w.shape]  # nothing of x where no weight asks
    dx = torch.autograd.grad(y.sum(), xr)[0]
    assert torch.allclose(dx, w.sum(0).expand(30, 64), atol=1e-4)
    br = b.clone().requires_grad_()
    db = torch.autograd.grad(linear8(x, w, br).sum(), br)[0]
    assert torch.allclose(db, torch.full((8,), 30.0, device=device))
    wr = w.clone().requires_grad_()
    kept.clear()
    with watch:
        y = linear8(x, wr, b)
    assert {t.dtype for t in kept if t.shape != w.shape} == {torch.int8, torch.uint8} and len(kept) == 3
    with torch.no_grad():
        assert linear8(x, wr, b).grad_fn is None


@pytest.mark.parametrize("device", DEVICES)
def test_linear8_bias_of_another_type(device):
    """16-bit weights beside a 32-bit bias: its gradient is not rounded to 16 bits."""
    x = torch.randn(300, 40, device=device).to(torch.bfloat16)
    w = torch.randn(24, 40, device=device).to(torch.bfloat16).requires_grad_()
    b = torch.randn(24, device=device, requires_grad=True)
    dy = torch.randn(300, 24, device=device).to(torch.bfloat16)
    dw, db = torch.autograd.grad(linear8(x, w, b), (w, b), dy)
    assert dw.dtype == torch.bfloat16 and db.dtype == torch.float32
    d = dy.cpu().double()
    close(db, d.sum(0), d.abs().sum(0), 300, "db")


@pytest.mark.parametrize("device", DEVICES)
def test_linear8_under_autocast(device):
    kind = torch.device(device).type
    x = torch.randn(20, 40, device=device, requires_grad=True)
    w = torch.randn(12, 40, device=device, requires_grad=True)
    with torch.autocast(kind, dtype=torch.bfloat16):
        y = linear8(x, w)
    assert y.dtype == torch.bfloat16
    dx, dw = torch.autograd.grad(y.float().sum(), (x, w))
    assert dx.dtype == torch.float32 and dw.dtype == torch.float32
    want = kept8(x.to(torch.bfloat16)).sum(0).expand(12, 40)
    close(dw, want, kept8(x.to(torch.bfloat16)).abs().sum(0).expand(12, 40), 20, "dw")


@pytest.mark.parametrize("device", DEVICES)
def test_linear8_no_gradient_of_the_gradient(device):
    x = torch.randn(4, 6, device=device, requires_grad=True)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(linear8(x, torch.randn(3, 6, device=device)).sum(), x, create_graph=True)


# ------------------------------------------------------------- the block, together
def block(x, w_in, b_in, w_out, b_out, dim, h0):
    p = linear8(x, w_in, b_in)
    y, last = gated_scan(p, dim, h0, keep="int8")
    return linear8(y, w_out, b_out), last


@pytest.mark.parametrize("device", DEVICES)
def test_block_trains(device):
    """Projection, scan and projection with every activation in 8 bits: gradients
    are near those that nothing was kept in 8 bits for."""
    g = torch.Generator().manual_seed(9)
    B, T, F, D = 4, 70, 20, 36
    x = torch.randn(B, T, F, generator=g).to(device)
    params = [torch.randn(3 * D, F, generator=g) / F**0.5, torch.randn(3 * D, generator=g) * 0.1,
              torch.randn(F, D, generator=g) / D**0.5, torch.zeros(F)]
    params = [t.to(device).requires_grad_() for t in params]
    h0 = torch.zeros(B, D, device=device)
    out, last = block(x, *params, D, h0)
    grads = torch.autograd.grad((out - x).square().mean(), params)

    p = torch.nn.functional.linear(x, params[0], params[1])
    h, ys = h0, []
    for t in range(T):
        f = torch.sigmoid(p[:, t, D : 2 * D])
        h = f * h + (1 - f) * p[:, t, :D]
        ys.append(h * torch.nn.functional.silu(p[:, t, 2 * D :]))
    ref = torch.nn.functional.linear(torch.stack(ys, 1), params[2], params[3])
    assert torch.allclose(out, ref, atol=1e-4) and torch.allclose(last, h, atol=1e-4)
    want = torch.autograd.grad((ref - x).square().mean(), params)
    for got, w in zip(grads, want):
        # a kept value is within 2^-7 of its group's largest, some 2.5 deviations:
        # under a sixtieth of a deviation a factor, three factors at most, and signs average
        assert float((got - w).norm() / w.norm()) < 0.05


@pytest.mark.parametrize("device", DEVICES)
def test_wide_lstm_keeps_its_inputs_in_8_bits(device):
    """The wide-LSTM path under ``checkpoint8``: the same outputs, gradients near
    the full ones, and no window in more than 8 bits between the two passes."""
    from gordo_amd.model.factories.lstm_autoencoder import lstm_symmetric
    from gordo_amd.ops.wide_lstm import wide_forward

    module = lstm_symmetric(n_features=12, dims=[40], lookback_window=9).to(device)
    w = torch.randn(6, 9, 12, device=device)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        out = wide_forward(module, w, checkpoint8=True)
    full = wide_forward(module, w)
    assert torch.allclose(out, full, atol=1e-5)
    assert not any(t.is_floating_point() and t.numel() in (6 * 9 * 12, 6 * 9 * 40) for t in kept)
    params = list(module.parameters())
    got = torch.autograd.grad(out.square().mean(), params)
    for g, f in zip(got, torch.autograd.grad(full.square().mean(), params)):
        assert float((g - f).norm() / f.norm()) < 0.05  # a kept value is within 2^-7 of its group's largest


@pytest.mark.gpu
def test_wide_lstm_estimator_trains_from_8_bits():
    """A width that no fused cell covers, from the estimator's own arguments, captured."""
    import numpy as np

    from gordo_amd.model.models import TorchLSTMAutoEncoder

    X = np.random.default_rng(0).normal(size=(60, 10)).astype(np.float32)
    model = TorchLSTMAutoEncoder(kind="lstm_symmetric", dims=[260], lookback_window=6, epochs=1, batch_size=16, seed=0, checkpoint8=True)
    model.fit(X)
    assert model.history["engine"] == "wide_lstm_gemmloop_graph"
    assert np.isfinite(model.history["loss"]).all() and np.isfinite(model.predict(X)).all()


@pytest.mark.gpu
def test_linear8_captured():
    g = torch.Generator().manual_seed(4)
    N, F, O = 3000, 70, 50
    x, w, b, dy = (torch.randn(*s, generator=g).to(torch.bfloat16).cuda() for s in ((N, F), (O, F), (O,), (N, O)))

    def work():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = linear8(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy), load8(save8(x)))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in range(3):
        for t in (x, dy):
            t.copy_(torch.randn(t.shape, generator=g))
        want = work()
        graph.replay()
        torch.cuda.synchronize()
        for a, b_ in zip(out, want):
            assert torch.equal(a, b_)


@pytest.mark.gpu
@pytest.mark.parametrize("frozen", [False, True], ids=["32-bit bias", "frozen weight"])
def test_linear8_bias_gradient_captured(frozen):
    g = torch.Generator().manual_seed(10)
    N, F, O = 5000, 70, 300
    x, w, dy = (torch.randn(*s, generator=g).to(torch.bfloat16).cuda() for s in ((N, F), (O, F), (N, O)))
    b = torch.randn(O, generator=g).cuda()

    def work():
        leaves = [t.detach().requires_grad_() for t in ((x, b) if frozen else (x, b, w))]
        y = linear8(leaves[0], w if frozen else leaves[2], leaves[1])
        return torch.autograd.grad(y, leaves, dy)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for _ in range(4):
        for t in (x, dy):
            t.copy_(torch.randn(t.shape, generator=g))
        want = work()
        graph.replay()
        torch.cuda.synchronize()
        for a, b_ in zip(out, want):
            assert torch.equal(a, b_)
        d = dy.cpu().double()
        close(out[1], d.sum(0), d.abs().sum(0), N, "db")


@pytest.mark.gpu
def test_save8_beyond_32_bits():
    """More than 2^31 values."""
    N, F = 2**20 + 3, 2080
    x = torch.zeros(N, F, dtype=torch.bfloat16, device="cuda")
    tail = values(7, F, torch.bfloat16, "cuda")
    x[-7:] = tail
    saved = save8(x)
    got = load8(saved)
    assert torch.equal(got[-7:].double().cpu(), kept8(tail)) and not got[:-7].any()


@pytest.mark.gpu
def test_weight_gradient_beyond_32_bits():
    """More than 2^31 values of dy, and of codes."""
    N, O, F = 2**20 + 3, 2080, 2080
    dy = torch.zeros(N, O, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(N, F, dtype=torch.bfloat16, device="cuda")
    dy[-7:], x[-7:] = torch.randn(7, O), torch.randn(7, F)
    dw, db = weight_grad8(dy, save8(x), bias=True, dtype=torch.float32)
    d, q = dy[-7:].cpu().double(), kept8(x[-7:])
    close(dw, d.t() @ q, d.abs().t() @ q.abs(), 7, "dw")
    close(db, d.sum(0), d.abs().sum(0), 7, "db")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N", [70, 3001])
def test_weight_gradient_of_infinite_dy(device, dtype, N):
    """What a scaled loss has overflowed to: infinite sums are infinite, of the sign that they
    have, in 32 bits as in 16; a NaN of any bits is none."""
    inf = float("inf")
    dy = torch.randn(N, 20).to(dtype)
    x = torch.rand(N, 40) + 0.5
    dy[5, 1], dy[9, 2], dy[60, 3] = inf, -inf, float("nan")
    dy[5, 4], dy[9, 4] = inf, -inf
    if dtype == torch.float32:
        dy[7, 6] = torch.tensor(0x7F800001, dtype=torch.int32).view(torch.float32)  # in its low half alone
    dy, x = dy.to(device), x.to(dtype).to(device)
    dw, db = weight_grad8(dy, save8(x), bias=True)
    for got in (dw, db[:, None]):
        assert (got[1] == inf).all() and (got[2] == -inf).all() and got[3].isnan().all() and got[4].isnan().all()
        assert got[0].isfinite().all() and got[7:].isfinite().all()
        assert got[6].isnan().all() if dtype == torch.float32 else got[6].isfinite().all()
    b = torch.zeros(20, dtype=dtype, device=device, requires_grad=True)
    w = torch.randn(20, 40, device=device).to(dtype)
    frozen = torch.autograd.grad(linear8(x, w, b), b, dy)[0]
    assert same(frozen.isfinite().float(), db.isfinite().float()) and (frozen[1] == inf).all()


@pytest.mark.parametrize("device", DEVICES)
def test_wide_lstm_makes_no_codes_of_windows_that_stay(device):
    """A training loop holds its windows through the backward pass: codes beside them would
    be bytes more, not fewer. The layers behind keep codes of what they read."""
    from gordo_amd.model.factories.lstm_autoencoder import lstm_symmetric
    from gordo_amd.ops.wide_lstm import wide_forward

    module = lstm_symmetric(n_features=12, dims=[40, 36], lookback_window=9).to(device)
    w = torch.randn(6, 9, 12, device=device)

    def kept_by(**how):
        kept = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
            out = wide_forward(module, w, **how)
        codes = sorted(t.numel() for t in kept if t.dtype == torch.int8)
        stays = any(t.untyped_storage().data_ptr() == w.untyped_storage().data_ptr() for t in kept)
        return out, codes, stays

    out, codes, stays = kept_by(checkpoint8=True, windows_stay=True)
    full, none, _ = kept_by()
    rows = 6 * 9
    assert codes == sorted(rows * n for n in (64, 64, 64)) and stays and not none  # 40, 36 and 36 wide, padded to 64
    assert torch.allclose(out, full, atol=1e-5)
    assert kept_by(checkpoint8=True)[1] == sorted(rows * n for n in (32, 64, 64, 64))
    first = [p for p in module.cells[-1].parameters()]
    assert all(g.isfinite().all() for g in torch.autograd.grad(out.square().mean(), first))


def test_checkpoint8_without_effect_is_said(caplog):
    """On estimators that have no such layers, and on the CPU, the argument changes nothing."""
    import logging

    import numpy as np

    from gordo_amd.model.models import TorchAutoEncoder, TorchLSTMAutoEncoder

    X = np.random.default_rng(0).normal(size=(40, 4)).astype(np.float32)
    dense = dict(kind="feedforward_symmetric", dims=[4], funcs=["tanh"], epochs=1, device="cpu")
    lstm = dict(kind="lstm_symmetric", dims=[4], funcs=["tanh"], lookback_window=3, epochs=1, device="cpu")
    for model, args in ((TorchAutoEncoder, dense), (TorchLSTMAutoEncoder, lstm)):
        with caplog.at_level(logging.WARNING):
            model(**args).fit(X)
            assert "checkpoint8" not in caplog.text
            model(**args, checkpoint8=True).fit(X)
            assert "checkpoint8 has no effect" in caplog.text
        caplog.clear()


@pytest.mark.gpu
def test_checkpoint8_without_effect_is_said_of_fused_engines(caplog):
    import logging

    import numpy as np

    from gordo_amd.model.models import TorchAutoEncoder, TorchLSTMAutoEncoder

    X = np.random.default_rng(0).normal(size=(300, 10)).astype(np.float32)
    with caplog.at_level(logging.WARNING):
        TorchAutoEncoder(kind="feedforward_hourglass", epochs=1, checkpoint8=True).fit(X)
        assert "checkpoint8 has no effect" in caplog.text
        caplog.clear()
        TorchLSTMAutoEncoder(kind="lstm_symmetric", dims=[16], lookback_window=6, epochs=1, batch_size=16, checkpoint8=True).fit(X)
        assert "checkpoint8 has no effect" in caplog.text
        caplog.clear()
        TorchLSTMAutoEncoder(kind="lstm_symmetric", dims=[260], lookback_window=6, epochs=1, batch_size=16, checkpoint8=True).fit(X[:40])
        assert "checkpoint8" not in caplog.text
