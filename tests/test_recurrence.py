"""Gated linear recurrence (ops.recurrence) against its definition in 64 bits.

Tolerances: an output of type t is off by its rounding, eps(t)/2 of the value,
and by the 32-bit arithmetic before it. A gate's relative error is at most
2^-20 (exp and reciprocal of an argument below 16 in magnitude); one token adds
that much of k (x - h) and two roundings of h, and errors are never amplified
(f <= 1), so after T tokens a state is off by at most 2^-20 M + T 2^-22 M, M
being the largest magnitude that takes part. The gradient's recursion is the
same one; its products of three to five such factors are allowed four times that.
"""
import pytest
import torch

from gordo_amd.ops import gated_scan, gated_step

EVERY = 16
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


# ------------------------------------------------------------------ definition
def kept8(v):
    """[..., D] in float64 as 8-bit codes keep it."""
    out = torch.empty_like(v)
    for at in range(0, v.shape[-1], 32):
        w = v[..., at : at + 32]
        _, e = torch.frexp(w.abs().amax(-1, keepdim=True))
        step = torch.exp2((e - 7).clamp_min(-126).double())
        out[..., at : at + 32] = torch.clamp(torch.round(w / step), -127, 127) * step
    return out


def definition(p, dim, h0, lengths, dy, dh, keep="input"):
    """(y, h_last, dp, dh0) in float64 on the CPU, token by token."""
    p, dy, dh = (t.detach().cpu().double() for t in (p, dy, dh))
    B, T, width = p.shape
    h = torch.zeros(B, dim, dtype=torch.float64) if h0 is None else h0.detach().cpu().double()
    n = torch.full((B, 1), T) if lengths is None else lengths.cpu().long().clamp(0, T)[:, None]
    y, dp = torch.zeros(B, T, dim, dtype=torch.float64), torch.zeros_like(p)
    states = []
    for t in range(T):
        states.append(h)
        x, f = p[:, t, :dim], torch.sigmoid(p[:, t, dim : 2 * dim])
        h = torch.where(t < n, f * h + (1 - f) * x, h)
        out = h
        if width == 3 * dim:
            z = p[:, t, 2 * dim :]
            out = h * z * torch.sigmoid(z)
        y[:, t] = torch.where(t < n, out, 0.0)
    last, q = h, p
    if keep == "int8":
        q = torch.cat([kept8(part) for part in p.split(dim, -1)], -1)
        for t in range(T):
            if t % EVERY:
                f = torch.sigmoid(q[:, t - 1, dim : 2 * dim])
                states[t] = f * states[t - 1] + (1 - f) * q[:, t - 1, :dim]
    c = dh
    for t in range(T - 1, -1, -1):
        x, f = q[:, t, :dim], torch.sigmoid(q[:, t, dim : 2 * dim])
        g, parts = dy[:, t], []
        if width == 3 * dim:
            z = q[:, t, 2 * dim :]
            s = torch.sigmoid(z)
            parts = [g * (f * states[t] + (1 - f) * x) * (s + z * s * (1 - s))]
            g = g * z * s
        g = g + c
        parts = [g * (1 - f), g * (states[t] - x) * f * (1 - f)] + parts
        dp[:, t] = torch.where(t < n, torch.cat(parts, -1), 0.0)
        c = torch.where(t < n, g * f, c)
    return y, last, dp, c


def inputs(B, T, D, dtype, device, gate=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    parts = 3 if gate else 2
    p = torch.randn(B, T, parts, D, generator=g)
    p[:, :, 1] = p[:, :, 1] * 1.5 + 1
    p = p.reshape(B, T, parts * D).to(dtype)
    h0, dh = torch.randn(B, D, generator=g), torch.randn(B, D, generator=g)
    dy = torch.randn(B, T, D, generator=g).to(dtype)
    return [t.to(device) for t in (p, h0, dy, dh)]


def near(got, want, scale, T, what, wide=1.0):
    got, want = got.detach().cpu(), want
    assert got.shape == want.shape, what
    eps = torch.finfo(got.dtype).eps
    allowed = eps / 2 * want.abs() * 1.0001 + wide * scale * (2.0**-20 + T * 2.0**-22)
    if got.dtype == torch.float16:
        allowed = allowed + 2.0**-25  # half a step of the subnormal numbers
    off = (got.double() - want).abs() - allowed
    assert torch.isfinite(got).all(), what
    assert off.max() <= 0 if off.numel() else True, (what, float(off.max()))


def check(p, D, h0, lengths, dy, dh, keep="input"):
    p = p.detach().requires_grad_()
    h = None if h0 is None else h0.detach().requires_grad_()
    y, last = gated_scan(p, D, h, lengths, keep=keep)
    leaves = (p,) if h is None else (p, h)
    grads = torch.autograd.grad((y, last), leaves, (dy, dh))
    want = definition(p, D, h0, lengths, dy, dh, keep)
    assert y.dtype == p.dtype and last.dtype == torch.float32
    T = p.shape[1]
    m = max(1.0, *(float(t.abs().max()) for t in (want[1], p.detach().double().cpu().nan_to_num(0)) if t.numel()))
    mg = max(1.0, *(float(t.abs().max()) for t in want[2:] if t.numel()))
    near(y, want[0], m * m, T, "y")
    near(last, want[1], m, T, "h_last")
    near(grads[0], want[2], 4 * m * m * mg, T, "dp")
    if h is not None:
        near(grads[1], want[3], mg, T, "dh0")
    return y, last, grads


# ----------------------------------------------------------------------- the scan
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("gate", [True, False], ids=["gate", "plain"])
@pytest.mark.parametrize("keep", ["input", "int8"])
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (3, 15, 2), (2, 16, 33), (2, 17, 64), (5, 49, 25), (1, 144, 50), (2, 129, 130)])
def test_scan_and_gradient(device, dtype, gate, keep, B, T, D):
    p, h0, dy, dh = inputs(B, T, D, dtype, device, gate)
    check(p, D, h0, None, dy, dh, keep)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("keep", ["input", "int8"])
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize("D", [7, 40])
def test_lengths_leave_padding_alone(device, keep, index, D):
    """Empty and full sequences, lengths outside the range, and padding that holds NaN and infinities."""
    T = 37
    p, h0, dy, dh = inputs(8, T, D, torch.bfloat16, device)
    lengths = torch.tensor([0, 1, 15, 16, 17, T, T + 100, -3], dtype=index)
    for b, n in enumerate([0, 1, 15, 16, 17, T, T, 0]):
        p[b, n:, ::2] = float("nan")
        p[b, n:, 1::2] = float("-inf")
        dy[b, n:] = float("inf")
    y, last, (dp, dh0) = check(p, D, h0, lengths.to(device), dy, dh, keep)
    assert not y[0].any() and not dp[0].any() and not y[2, 15:].any() and not dp[2, 15:].any()
    assert torch.equal(last[0], h0[0]) and torch.equal(last[7], h0[7]) and torch.equal(dh0[0], dh[0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_padding_of_zeros_is_a_longer_batch(device, dtype):
    p, h0, dy, dh = inputs(3, 40, 10, dtype, device)
    lengths = torch.full((3,), 25, device=device)
    y, last = gated_scan(p, 10, h0, lengths)
    short, short_last = gated_scan(p[:, :25].contiguous(), 10, h0)
    assert torch.equal(y[:, :25], short) and torch.equal(last, short_last)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("first,extra", [(0, 6), (4, 4), (1, 5), (3, 8)])
def test_strides(device, first, extra):
    """A slice of a wider buffer, at even and odd places, time and batch swapped."""
    B, T, D = 3, 35, 12
    p, h0, dy, dh = inputs(B, T, D, torch.bfloat16, device)
    wide = torch.full((T, B, first + 3 * D + extra), 9.0, dtype=p.dtype, device=device)
    view = wide[:, :, first : first + 3 * D].transpose(0, 1)
    view.copy_(p)
    dyw = torch.full((B, T, D + extra), 9.0, dtype=p.dtype, device=device)[..., extra:]
    dyw.copy_(dy)
    a = check(view, D, h0, None, dyw, dh)
    b = check(p, D, h0, None, dy, dh)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2][0], b[2][0])
    turned = p.transpose(1, 2).contiguous().transpose(1, 2)  # last axis not of unit stride
    assert torch.equal(gated_scan(turned, D, h0)[0], b[0])


@pytest.mark.parametrize("device", DEVICES)
def test_parts_of_the_gradient(device):
    """Only y, only h_last, an expanded gradient, a projection alone, no h0."""
    B, T, D = 2, 33, 6
    p, h0, dy, dh = inputs(B, T, D, torch.float32, device)
    check(p, D, None, None, dy, dh)
    check(p, D, h0, None, torch.ones((), device=device).expand(B, T, D), torch.zeros_like(dh))
    q = p.clone().requires_grad_()
    only_last = torch.autograd.grad(gated_scan(q, D, h0)[1].sum(), q)[0]
    want = definition(p, D, h0, None, torch.zeros_like(dy), torch.ones_like(dh))[2]
    near(only_last, want, 40.0, T, "dp of h_last")
    h = h0.clone().requires_grad_()
    dh0 = torch.autograd.grad(gated_scan(p, D, h)[0].sum(), h)[0]
    want = definition(p, D, h0, None, torch.ones_like(dy), torch.zeros_like(dh))[3]
    near(dh0, want, 40.0, T, "dh0 of y")


@pytest.mark.parametrize("keep", ["input", "int8"])
@pytest.mark.parametrize("gate", [True, False])
def test_definition_against_differences(gate, keep):
    """The formula of the gradient is the derivative of the formula of the scan
    (with codes: where nothing is lost, that is at values that codes hold)."""
    B, T, D = 2, 5, 3
    p, h0, dy, dh = inputs(B, T, D, torch.float32, "cpu", gate)
    p = kept8(p.double().reshape(B, T, -1, D)).reshape(B, T, -1)
    y, last, dp, dh0 = definition(p, D, h0, None, dy, dh, keep)
    loss = lambda p, h: sum(float((a * b.double()).sum()) for a, b in zip(definition(p, D, h, None, dy, dh)[:2], (dy, dh)))  # noqa: E731
    step = 1e-5  # central differences: error step^2 and 1e-16 / step
    g = torch.Generator().manual_seed(3)
    for _ in range(6):
        v, w = torch.randn(p.shape, generator=g, dtype=torch.float64), torch.randn(h0.shape, generator=g, dtype=torch.float64)
        slope = (loss(p + step * v, h0.double() + step * w) - loss(p - step * v, h0.double() - step * w)) / (2 * step)
        assert abs(slope - float((dp * v).sum() + (dh0 * w).sum())) < 1e-7 * max(1.0, abs(slope))


@pytest.mark.parametrize("device", DEVICES)
def test_long_memory_keeps_its_digits(device):
    """k = 2^-20: 1 - k has five bits of it in 32 bits, the scan all of them."""
    r = 13.862942695617676  # log(2^20 - 1)
    T, D = 512, 4
    p = torch.zeros(1, T, 2 * D, device=device)
    p[..., :D], p[..., D:] = 1.0, r
    y, last = gated_scan(p, D)
    k = torch.sigmoid(-torch.tensor(r, dtype=torch.float64))
    want = 1 - (1 - k) ** T  # h after T tokens of x = 1
    # a gate is off by 2^-20 of itself, each of T updates rounds h, which is below 2^-10
    assert (last.double().cpu() - want).abs().max() < 2.0**-20 * want + T * 2.0**-35


@pytest.mark.parametrize("device", DEVICES)
def test_extreme_gates(device):
    """Gates that are wide open or shut pass or hold the state exactly."""
    p = torch.zeros(1, 40, 6, device=device)
    p[..., :2] = torch.arange(40.0, device=device)[:, None]
    p[..., 2], p[..., 3] = 200.0, -200.0
    p[..., 4:] = 1.0
    h0 = torch.tensor([[5.0, 7.0]], device=device)
    y, last = gated_scan(p[..., :4].contiguous(), 2, h0)
    assert (y[..., 0] == 5).all() and torch.equal(y[0, :, 1].cpu(), torch.arange(40.0))
    p[..., 2], p[..., 3] = float("inf"), float("-inf")
    y, last = gated_scan(p[..., :4].contiguous(), 2, h0)
    assert (y[..., 0] == 5).all() and torch.equal(y[0, :, 1].cpu(), torch.arange(40.0))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,D", [(3, 6), (40, 6), (40, 130), (1500, 64)])
def test_overflowed_state_passes_padding(device, T, D):
    """An infinite state is what it is behind a sequence's last token, and so is a
    start state where there is no token at all."""
    inf = float("inf")
    p = torch.zeros(3, T, 2 * D, device=device)
    p[1, 1, :D] = inf  # the last token of this one
    p[:, 2:] = float("nan")
    h0 = torch.tensor([inf, 1.0, -2.0], device=device)[:, None].expand(3, D)
    y, last = gated_scan(p, D, h0, torch.tensor([0, 2, 1], device=device))
    assert (last[0] == inf).all() and (last[1] == inf).all() and (last[2] == -1.0).all()
    assert not y[0].any() and (y[1, 0] == 0.5).all() and (y[1, 1] == inf).all() and not y[1, 2:].any()


def test_default_types_are_not_asked():
    p = torch.randn(2, 5, 12)
    want = gated_scan(p, 4)
    try:
        torch.set_default_dtype(torch.float64)
        got = gated_scan(p, 4)
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("device", DEVICES)
def test_step_tells_graphs_that_the_state_changed(device):
    state = torch.ones(2, 4, device=device)
    w = torch.ones(2, 4, device=device, requires_grad=True)
    kept = (state * w).sum()
    with torch.no_grad():
        gated_step(torch.randn(2, 12, device=device), state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
    with torch.inference_mode():
        state = torch.ones(2, 4, device=device)
        assert gated_step(torch.randn(2, 12, device=device), state).isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
def test_empty(device):
    h0 = torch.randn(2, 3, device=device)
    y, last = gated_scan(torch.randn(2, 0, 9, device=device), 3, h0)
    assert y.shape == (2, 0, 3) and torch.equal(last, h0)
    y, last = gated_scan(torch.randn(0, 4, 6, device=device), 3)
    assert y.shape == (0, 4, 3) and last.shape == (0, 3)


def test_scan_refuses():
    p = torch.randn(2, 4, 9)
    for bad in (
        lambda: gated_scan(p.double(), 3),
        lambda: gated_scan(p.to(torch.int32), 3),
        lambda: gated_scan(p[0], 3),
        lambda: gated_scan(p, 4),
        lambda: gated_scan(p, 9),
        lambda: gated_scan(p, 0),
        lambda: gated_scan(p, 3.0),
        lambda: gated_scan(p, 3, torch.randn(2, 3).double()),
        lambda: gated_scan(p, 3, torch.randn(3, 2)),
        lambda: gated_scan(p, 3, torch.randn(1, 3)),
        lambda: gated_scan(p, 3, lengths=torch.tensor([1.0, 2.0])),
        lambda: gated_scan(p, 3, lengths=torch.tensor([1])),
        lambda: gated_scan(p, 3, lengths=[1, 2]),
        lambda: gated_scan(p, 3, h0=torch.randn(2, 3, device="meta")),
        lambda: gated_scan(p, 3, keep="fp8"),
    ):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("device", DEVICES)
def test_no_gradient_of_the_gradient(device):
    p = torch.randn(1, 4, 6, device=device, requires_grad=True)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(gated_scan(p, 3)[0].sum(), p, create_graph=True)


# ----------------------------------------------------------------------- the step
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("gate", [True, False], ids=["gate", "plain"])
@pytest.mark.parametrize("B,D", [(1, 1), (3, 50), (2, 255), (4, 1030)])
def test_steps_are_the_scan(device, dtype, gate, B, D):
    """Token by token, the step gives what the scan gives, and the scan's state goes on in it."""
    T = 5
    p, h0, dy, dh = inputs(B, T, D, dtype, device, gate)
    want = definition(p, D, h0, None, dy, dh)
    state = h0.clone()
    for t in range(T):
        y = gated_step(p[:, t], state)
        near(y, want[0][:, t], 25.0, T, "y")
    near(state, want[1], 5.0, T, "state")
    state = gated_scan(p[:, :3], D, h0)[1]
    gated_step(p[:, 3], state)
    near(gated_step(p[:, 4], state), want[0][:, 4], 25.0, T, "y after a scan")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize("apart", [False, True], ids=["in place", "out"])
def test_slots(device, index, apart):
    """Padding rows, slots that come again, and slots that no row names."""
    S, D = 9, 70
    slots = torch.tensor([4, -1, 7, 4, 2, S, 4, -(2**31), 7, 2**31 - 1], dtype=index)
    p, _, _, _ = inputs(len(slots), 1, D, torch.float32, device)
    p = p[:, 0]
    before = torch.randn(S, D, generator=torch.Generator().manual_seed(1)).to(device)
    state = before.clone()
    out = torch.full_like(state, 3.0) if apart else None
    y = gated_step(p, state, slots.to(device), out=out)
    want = before.cpu().double()
    for b, s in enumerate(slots.tolist()):
        if not 0 <= s < S:
            assert not y[b].any()
            continue
        x, r, z = p[b].cpu().double().split(D)
        f = torch.sigmoid(r)
        want[s] = f * want[s] + (1 - f) * x
        near(y[b], want[s] * z * torch.sigmoid(z), 25.0, 3, f"y of row {b}")
    named = torch.tensor(sorted({s for s in slots.tolist() if 0 <= s < S}))
    rest = torch.tensor([s for s in range(S) if s not in named.tolist()])
    got = state if out is None else out
    near(got.cpu()[named], want[named], 5.0, 3, "states")
    assert torch.equal(state.cpu()[rest], before.cpu()[rest])
    if apart:
        assert (out.cpu()[rest] == 3.0).all() and torch.equal(state, before)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize("first", [0, 1])
def test_many_rows_share_slots(device, index, first):
    """Several tokens of many streams in one call, slots at any address: as token after token."""
    B, S, D = 403, 150, 34
    g = torch.Generator().manual_seed(8)
    p = inputs(B, 1, D, torch.float32, "cpu")[0][:, 0]
    slots = torch.randint(-5, S + 5, (B + first,), generator=g, dtype=index)[first:]
    state = torch.randn(S, D, generator=g)
    want, ys = state.double(), torch.zeros(B, D, dtype=torch.float64)
    for b, s in enumerate(slots.tolist()):
        if 0 <= s < S:
            x, r, z = p[b].double().split(D)
            want[s] = torch.sigmoid(r) * want[s] + torch.sigmoid(-r) * x
            ys[b] = want[s] * z * torch.sigmoid(z)
    on = slots.to(device)
    if first:  # .to() makes a buffer of its own: put it at an odd place again
        on = torch.cat([on[:first], on])[first:]
    state = state.to(device)
    y = gated_step(p.to(device), state, on)
    near(y, ys, 25.0, 20, "y")
    near(state, want, 5.0, 20, "state")


@pytest.mark.parametrize("device", DEVICES)
def test_step_of_nothing(device):
    state = torch.randn(3, 4, device=device)
    assert gated_step(torch.randn(0, 8, device=device), state, torch.zeros(0, dtype=torch.int32, device=device)).shape == (0, 4)
    none = torch.empty(0, 4, device=device)
    assert not gated_step(torch.randn(2, 8, device=device), none, torch.zeros(2, dtype=torch.int64, device=device)).any()


def test_step_refuses():
    p, state = torch.randn(2, 9), torch.randn(5, 3)
    slots = torch.tensor([0, 1])
    big = torch.randn(11, 3)
    for bad in (
        lambda: gated_step(p.double(), state, slots),
        lambda: gated_step(p[:, :8], state, slots),
        lambda: gated_step(p[None], state, slots),
        lambda: gated_step(p, state.half(), slots),
        lambda: gated_step(p, state.t().contiguous().t(), slots),
        lambda: gated_step(p, state[0], slots),
        lambda: gated_step(p, state),
        lambda: gated_step(p, state, slots.float()),
        lambda: gated_step(p, state, slots[:1]),
        lambda: gated_step(p, state, torch.zeros(2, dtype=torch.int32, device="meta")),
        lambda: gated_step(p, state, slots, out=torch.randn(4, 3)),
        lambda: gated_step(p, state, slots, out=state.half()),
        lambda: gated_step(p, big[:5], slots, out=big[1:6]),
        lambda: gated_step(p.requires_grad_(), state, slots),
    ):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------- on the GPU alone
@pytest.mark.gpu
@pytest.mark.parametrize("keep", ["input", "int8"])
@pytest.mark.parametrize("gate", [True, False], ids=["gate", "plain"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize(
    "B,T,D",
    [
        (1, 513, 64),     # time split over blocks that are chained
        (1, 2049, 40),    # the chain's first link, forward, and a lone token behind it
        (2, 5000, 33),    # many links, lanes that straddle two sequences
        (1, 4097, 1),     # one channel
        (5, 1100, 130),
        (4, 2300, 200),   # links of 16 tiles, forward too
        (3, 4, 130),      # short tiles
        (50, 2, 64),
        (40000, 1, 66),
        (700, 150, 50),   # a block walks several tiles
        (600, 650, 120),  # many of them
        (2200, 70, 62),   # a wave walks alone
        (70000, 3, 4),    # a tile is more than a sequence
        (9000, 37, 25),   # narrow rows, staged: runs at every 2-byte place
        (6000, 35, 50),
        (4500, 33, 33),   # a sequence a wave
        (3, 9, 130),      # a wave walks alone, row by row
        (2100, 40, 130),
        (2100, 33, 65),
        (4100, 21, 64),
    ],
)
def test_every_way_of_splitting(B, T, D, dtype, gate, keep):
    p, h0, dy, dh = inputs(B, T, D, dtype, "cuda", gate)
    lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(2)).cuda()
    lengths[-1] = T
    check(p, D, h0, lengths, dy, dh, keep)


@pytest.mark.gpu
@pytest.mark.parametrize("keep", ["input", "int8"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,T,D", [(7, 4, 2), (900, 3, 50), (5, 1, 62), (6, 11, 66), (3, 16, 126), (2700, 40, 100), (3, 2, 100)])
def test_pairs_of_channels_in_narrow_rows(B, T, D, dtype, keep):
    """16-bit rows that are whole words: as they lie, and with a word between sequences."""
    p, h0, dy, dh = inputs(B, T, D, dtype, "cuda")
    lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(3)).cuda()
    a = check(p, D, h0, lengths, dy, dh, keep)
    for first in (0, 1, 2):
        n = T * 3 * D
        buf = torch.full((B * (n + 2) + 2,), float("nan"), dtype=dtype, device="cuda")
        view = buf.as_strided((B, T, 3 * D), (n + 2, 3 * D, 1), first)
        view.copy_(p)
        b = check(view, D, h0, lengths, dy, dh, keep)
        assert torch.equal(a[0], b[0])


@pytest.mark.gpu
@pytest.mark.parametrize("first", [0, 1, 2, 3])
def test_narrow_rows_in_a_larger_buffer(first):
    """Dense sequences that start anywhere: what lies between them is left alone."""
    B, T, D = 7000, 20, 25
    p, h0, dy, dh = inputs(B, T, D, torch.bfloat16, "cuda", gate=False)
    n = T * 2 * D
    buf = torch.full((B, n + 3), float("nan"), dtype=p.dtype, device="cuda")
    view = buf.as_strided((B, T, 2 * D), (n + 3, 2 * D, 1), first)
    view.copy_(p)
    a, b = check(view, D, h0, None, dy, dh), check(p, D, h0, None, dy, dh)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2][0], b[2][0])


@pytest.mark.gpu
@pytest.mark.parametrize("T,D", [(3000, 32), (3000, 8192)])
def test_nan_goes_where_it_belongs(T, D):
    """A NaN of any bits in one channel of one token: that channel from there on,
    and its gradient up to there; the chain between blocks waits for no such word."""
    p, h0, dy, dh = inputs(1, T, D, torch.float32, "cuda", gate=False)
    p[0, 100, 5] = torch.tensor(-1, dtype=torch.int32).view(torch.float32)
    q = p.clone().requires_grad_()
    y, last = gated_scan(q, D, h0)
    bad = y[0].isnan()
    assert not bad[:100].any() and bad[100:, 5].all() and int(bad.sum()) == T - 100
    assert last[0, 5].isnan() and int(last.isnan().sum()) == 1
    dyn = dy.clone()
    dyn[0, T - 50, 7] = torch.tensor(-1, dtype=torch.int32).view(torch.float32)
    q = inputs(1, T, D, torch.float32, "cuda", gate=False)[0].requires_grad_()
    dp = torch.autograd.grad(gated_scan(q, D, h0), q, (dyn, dh))[0][0, :, :D].isnan()
    assert dp[: T - 49, 7].all() and int(dp.sum()) == T - 49


@pytest.mark.gpu
def test_same_inputs_same_bits():
    p, h0, dy, dh = inputs(2, 700, 96, torch.bfloat16, "cuda")
    lengths = torch.tensor([700, 433], device="cuda")
    runs = [check(p, 96, h0, lengths, dy, dh, "int8") for _ in range(3)]
    for y, last, (dp, dh0) in runs[1:]:
        assert torch.equal(y, runs[0][0]) and torch.equal(last, runs[0][1])
        assert torch.equal(dp, runs[0][2][0]) and torch.equal(dh0, runs[0][2][1])


@pytest.mark.gpu
def test_on_a_stream_of_its_own():
    p, h0, dy, dh = inputs(2, 100, 40, torch.float32, "cuda")
    want = check(p, 40, h0, None, dy, dh)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = check(p, 40, h0, None, dy, dh)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[2][0], want[2][0])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [30, 900, 6000])
def test_captured(T):
    """Forward, backward and step in a graph, replayed with eager work between."""
    D = 32
    p, h0, dy, dh = inputs(1, T, D, torch.bfloat16, "cuda")
    row, state = p[:, 0].clone(), h0.clone()

    def work(p, h0, dy, dh, row, state):
        p, h0 = p.detach().requires_grad_(), h0.detach().requires_grad_()
        y, last = gated_scan(p, D, h0, keep="int8")
        dp, dh0 = torch.autograd.grad((y, last), (p, h0), (dy, dh))
        with torch.no_grad():
            return y.detach(), last.detach(), dp, dh0, gated_step(row, state)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work(p, h0, dy, dh, row, state.clone())
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(p, h0, dy, dh, row, state)
    for seed in range(1, 4):
        fresh = inputs(1, T, D, torch.bfloat16, "cuda", seed=seed)
        for a, b in zip((p, h0, dy, dh, row, state), (*fresh, fresh[0][:, 0], fresh[1])):
            a.copy_(b)
        eager_state = state.clone()
        want = work(p.clone(), h0, dy, dh, row, eager_state)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*out, state), (*want, eager_state)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Two sequences more than 2^31 elements apart, tokens far apart too."""
    T, D = 20, 16
    p, h0, dy, dh = inputs(2, T, D, torch.bfloat16, "cuda")
    far = 2**31 + 64
    buf = torch.empty(far + (T - 1) * 2**20 + 3 * D, dtype=torch.bfloat16, device="cuda")
    view = buf.as_strided((2, T, 3 * D), (far, 2**20, 1))
    view.copy_(p)
    a, b = check(view, D, h0, None, dy, dh), check(p, D, h0, None, dy, dh)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2][0], b[2][0])


# ------------------------------------------ the digits of gates that hold and let go
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [37, 74, 1480])
def test_gates_keep_their_digits_at_both_ends(device, D):
    """f near 0 as k near 0: 1 - k has lost f's digits at r = -8, all of them at -18.

    One token, so every output is a product: dx = g k, dr = g (h0 - x) k f, dh0 = g f,
    and y = f h0 where x is 0. A gate is off by 2^-19 of itself (an argument of exp of
    up to 18 log2(e) = 26 is rounded by 2^-20, times log 2; exp, 1 + e, the reciprocal
    and the product some 2^-22 each), a product of two by twice that."""
    r = torch.linspace(-18, 18, 37).repeat(D // 37)
    x, h0 = torch.zeros(D), torch.full((D,), 3.0)
    p = torch.cat([x, r])[None, None].to(device).requires_grad_()
    h = h0[None].to(device).requires_grad_()
    y, last = gated_scan(p, D, h)
    dp, dh0 = torch.autograd.grad(last, (p, h), torch.full((1, D), 0.75, device=device))
    f, k = torch.sigmoid(r.double()), torch.sigmoid(-r.double())

    def relative(got, want, allowed):
        off = (got.detach().cpu().double().flatten() / want - 1).abs()
        assert float(off.max()) < allowed, (float(r[off.argmax()]), float(off.max()))

    relative(dh0, 0.75 * f, 2.0**-19)
    relative(dp[..., :D], 0.75 * k, 2.0**-19)
    relative(dp[..., D:], 0.75 * 3 * k * f, 2.0**-18)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,D", [(5, 33), (40, 37), (40, 130), (300, 74), (1500, 37)])
def test_one_token_lets_a_long_memory_go(device, T, D):
    """All gates hold but one, at another token for each channel: what passes is f of
    that one, also through the maps of tiles that are folded into each other."""
    r = torch.full((T, D), 30.0)  # f = 1 - 2^-43
    at = torch.randint(0, T, (D,), generator=torch.Generator().manual_seed(4))
    lets = torch.linspace(-18, -8, D)
    r[at, torch.arange(D)] = lets
    p = torch.cat([torch.zeros(T, D), r], 1)[None].to(device).requires_grad_()
    h = torch.full((1, D), 3.0, device=device, requires_grad=True)
    y, last = gated_scan(p, D, h)
    dp, dh0 = torch.autograd.grad(last, (p, h), torch.ones(1, D, device=device))
    f = torch.sigmoid(lets.double())
    # the other gates' products round to what they were: f of 1 - 2^-43 takes nothing away
    assert float((dh0[0].cpu().double() / f - 1).abs().max()) < 2.0**-19
    dr = dp[0, at, D + torch.arange(D)].cpu().double()
    assert float((dr / (3 * f * (1 - f)) - 1).abs().max()) < 2.0**-18


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,D", [(1, 37), (1, 74), (40, 37), (300, 74)])
def test_a_state_keeps_the_digits_of_what_is_let_go(device, T, D):
    """x = 0 throughout: a state is the product of the f before it, whatever their size."""
    r = torch.full((T, D), 30.0)
    lets = torch.linspace(-18, 18, 37).repeat(D // 37)
    r[T // 2] = lets
    p = torch.cat([torch.zeros(T, D), r], 1)[None].to(device)
    h0 = torch.full((1, D), 3.0, device=device)
    y, last = gated_scan(p, D, h0)
    want = 3 * torch.sigmoid(lets.double())
    assert float((last[0].cpu().double() / want - 1).abs().max()) < 2.0**-19
    assert torch.equal(y[0, -1], last[0])
    gated_step(p[:, T // 2], h0)
    assert float((h0[0].cpu().double() / want - 1).abs().max()) < 2.0**-19


# ------------------------------------------------------------- near the largest number
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("B,T,D", [(3, 1, 40), (2, 2, 66), (3, 40, 33), (2, 700, 64), (1, 40, 130)])
def test_states_between_the_largest_numbers(device, dtype, B, T, D):
    """x and h of opposite signs, further apart than the largest number: a state lies
    between them, and so does everything that is made of finite ones."""
    g = torch.Generator().manual_seed(5)
    top = torch.finfo(dtype).max
    x = (torch.rand(B, T, D, generator=g) * 2 - 1) * top
    x[:, ::3] = top
    x[:, 1::3] = -top
    p = torch.cat([x, torch.randn(B, T, D, generator=g) * 4], -1).to(dtype)
    h0 = ((torch.rand(B, D, generator=g) * 2 - 1) * torch.finfo(torch.float32).max)
    dy, dh = torch.randn(B, T, D, generator=g) * 2.0**-10, torch.randn(B, D, generator=g) * 2.0**-10
    dy = dy.to(dtype)
    want = definition(p, D, h0, None, dy, dh)
    p, h0 = p.to(device).requires_grad_(), h0.to(device).requires_grad_()
    y, last = gated_scan(p, D, h0)
    dp, dh0 = torch.autograd.grad((y, last), (p, h0), (dy.to(device), dh.to(device)))
    big = torch.finfo(torch.float32).max
    near(y, want[0], big, T, "y")
    near(last, want[1], big, T, "h_last")
    near(dp[..., D:], want[2][..., D:], big * float(want[3].abs().max() + want[2][..., :D].abs().max()), T, "dr")
    near(dh0, want[3], 0.1, T, "dh0")
    state = h0.detach().clone()
    with torch.no_grad():
        near(gated_step(p[:, 0], state), want[0][:, 0], big, 1, "y of a step")


@pytest.mark.parametrize("device", DEVICES)
def test_opposite_values_meet_half_way(device):
    x = torch.tensor([3e38, -3e38], device=device)
    p = torch.stack([x, torch.zeros_like(x)], 1)[None]
    y, last = gated_scan(p, 1)
    # half of 3e38 is 1.5e38, half of that and half of -3e38: -7.5e37, two roundings each
    assert abs(float(last) / -7.5e37 - 1) < 2.0**-20


# ------------------------------------------------------------------ infinite gradients
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gate", [True, False], ids=["gate", "plain"])
@pytest.mark.parametrize("keep", ["input", "int8"])
@pytest.mark.parametrize("T,D", [(3, 6), (40, 6), (40, 130), (300, 64), (1500, 64)])
def test_an_infinite_gradient_passes_padding(device, gate, keep, T, D):
    """A gradient that a scaled loss has overflowed is what it is in front of the padding,
    and is not taken for a number at the tokens before."""
    inf = float("inf")
    parts = 3 if gate else 2
    p = torch.zeros(4, T, parts * D, device=device)
    p[:, 2:] = float("nan")
    dh = torch.tensor([inf, -inf, inf, 1.0], device=device)[:, None].expand(4, D).contiguous()
    dy = torch.zeros(4, T, D, device=device)
    dy[3, 2:] = inf
    lengths = torch.tensor([0, 1, 2, 2], device=device)
    p.requires_grad_()
    h0 = torch.ones(4, D, device=device, requires_grad=True)
    dp, dh0 = torch.autograd.grad(gated_scan(p, D, h0, lengths, keep=keep), (p, h0), (dy, dh))
    # half gates: f = k = 1/2 at every token there is
    assert (dh0[0] == inf).all() and (dh0[1] == -inf).all() and (dh0[2] == inf).all() and (dh0[3] == 0.25).all()
    assert not dp[0].any() and not dp[1, 1:].any() and not dp[2:, 2:].any()
    assert (dp[1, 0, :D] == -inf).all() and (dp[2, :2, :D] == inf).all()
    assert (dp[3, :2, :D] == torch.tensor([0.25, 0.5], device=device)[:, None]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("B,T,D", [(2, 50, 20), (1, 50, 130), (1, 1200, 64)])
def test_what_follows_no_number_is_none(device, bad, B, T, D):
    """A state, or a gradient, that is not finite reaches all that depends on it."""
    p, h0, dy, dh = inputs(B, T, D, torch.float32, device, gate=False)
    at = T // 2
    q = p.clone()
    q[:, at, 3] = bad
    y, last = gated_scan(q, D, h0)
    assert not y[:, at:, 3].isfinite().any() and not last[:, 3].isfinite().any()
    assert y[:, :at].isfinite().all() and y[..., 4:].isfinite().all()
    dy[:, at, 3] = bad
    p.requires_grad_()
    h0.requires_grad_()
    dp, dh0 = torch.autograd.grad(gated_scan(p, D, h0), (p, h0), (dy, dh))
    assert not dp[:, : at + 1, 3].isfinite().any() and not dh0[:, 3].isfinite().any()
    assert dp[:, at + 1 :].isfinite().all() and dp[..., 4:D].isfinite().all()


# ---------------------------------------------------------------- calls with no answer
@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_is_refused(device):
    """A tangent is not dropped without a word: with and without gradients, of p and of h0."""
    fw = torch.autograd.forward_ad
    p, h0 = torch.randn(1, 4, 6, device=device), torch.randn(1, 3, device=device)
    with fw.dual_level():
        dual_p, dual_h = fw.make_dual(p, torch.ones_like(p)), fw.make_dual(h0, torch.ones_like(h0))
        for call in (lambda: gated_scan(dual_p, 3), lambda: gated_scan(p, 3, dual_h),
                     lambda: gated_scan(p.clone().requires_grad_(), 3, dual_h)):
            with pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward"):
                call()
            with torch.no_grad(), pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward"):
                call()
    assert gated_scan(p, 3, h0)[0].isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
def test_step_refuses_tangents(device):
    fw = torch.autograd.forward_ad
    p, state = torch.randn(2, 9, device=device), torch.randn(2, 3, device=device)
    kept = state.clone()
    with fw.dual_level():
        for make in (lambda: (fw.make_dual(p, torch.ones_like(p)), state, None),
                     lambda: (p, fw.make_dual(state, torch.ones_like(state)), None),
                     lambda: (p, state, fw.make_dual(state.clone(), torch.ones_like(state)))):
            q, s, out = make()
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="no gradient"):
                    gated_step(q, s, out=out)
    assert torch.equal(state, kept)
    gated_step(p, state)


@pytest.mark.parametrize("device", DEVICES)
def test_step_refuses_an_out_that_asks_for_a_gradient(device):
    """Overwritten in place, `out` would leave a graph with gradients of values that are gone."""
    p, state = torch.randn(2, 9, device=device), torch.randn(2, 3, device=device)
    w = torch.ones(2, 3, device=device, requires_grad=True)
    part, leaf = w * 2, torch.zeros(2, 3, device=device, requires_grad=True)
    for out in (part, leaf):
        kept = out.detach().clone()
        with pytest.raises(ValueError, match="no gradient"):
            gated_step(p, state, out=out)
        assert torch.equal(out, kept)
    with torch.no_grad():
        assert gated_step(p, state, out=leaf).isfinite().all() and leaf.any()


@pytest.mark.gpu
@pytest.mark.parametrize("keep", ["input", "int8"])
def test_bits_under_more_padding(keep):
    """How time is split follows from the padded length: where the split is the same, so are
    the bits; across its border (four tiles of 128 tokens in a block's walk, five and more
    in a chain of blocks) a sequence's results are near."""
    n, D = 500, 40
    p, h0, dy, dh = inputs(2, n, D, torch.float32, "cuda")
    want = definition(p, D, h0, None, dy, dh, keep)
    runs = {}
    for T in (n, 512, 513, 600, 640, 3000):
        wide = torch.full((2, T, 3 * D), float("nan"), device="cuda")
        wide_dy = torch.full((2, T, D), float("nan"), device="cuda")
        wide[:, :n], wide_dy[:, :n] = p, dy
        wide.requires_grad_()
        h = h0.clone().requires_grad_()
        y, last = gated_scan(wide, D, h, torch.full((2,), n, device="cuda"), keep=keep)
        dp, dh0 = torch.autograd.grad((y, last), (wide, h), (wide_dy, dh))
        runs[T] = y.detach()[:, :n], last.detach(), dp[:, :n], dh0
        m = float(p.abs().max())
        near(y[:, :n], want[0], m * m, n, "y")
        near(last, want[1], m, n, "h_last")
        near(dh0, want[3], 8.0, n, "dh0")
    for a, b in ((n, 512), (513, 600), (600, 640)):
        assert all(torch.equal(s, t) for s, t in zip(runs[a][:2], runs[b][:2]))


# --------------------------------------------------- every element by its own error bound
U = 2.0**-22  # four roundings of 2^-24: two of a token's update, two of the maps it goes through
GATE = 2.0**-20  # a gate's smaller factor, relative: exp and reciprocal of an argument below 16


def bounded(p, dim, h0, lengths, dy, dh, keep="input", seam=None):
    """((value, error) of y, h_last, dp and dh0): the definition beside the first-order errors
    of 32-bit arithmetic, token by token. M is a sum of magnitudes, E the error that it may
    carry; both fade with the gates, so a bound is as local as the memory. What is in it:

    - the smaller of f and k is off by GATE of itself, the other one by the same amount
    - a token's update of a state, or of the gradient's carry, by U of its magnitudes
    - silu by 2^-19 of itself (sigmoid 2^-20, products), silu' by 2^-18 of its two terms
    - products and differences of these by their factors' errors and U of their magnitudes

    ``seam``: the carry is lost in front of this token (a mistake for the test of the test)."""
    p, dy, dh = (t.detach().cpu().double() for t in (p, dy, dh))
    B, T, width = p.shape
    h = torch.zeros(B, dim, dtype=torch.float64) if h0 is None else h0.detach().cpu().double()
    n = torch.full((B, 1), T) if lengths is None else lengths.cpu().long().clamp(0, T)[:, None]
    q = p if keep == "input" else torch.cat([kept8(part) for part in p.split(dim, -1)], -1)

    def gates(p, t):
        r = p[:, t, dim : 2 * dim]
        return p[:, t, :dim], torch.sigmoid(r), torch.sigmoid(-r)

    def token(p, t, h, M, E):
        x, f, k = gates(p, t)
        live = t < n
        m = f * M + k * x.abs()
        e = f * E + GATE * torch.minimum(f, k) * (x.abs() + M) + U * m
        return torch.where(live, f * h + k * x, h), torch.where(live, m, M), torch.where(live, e, E)

    def gate_of(p, t):
        z = p[:, t, 2 * dim :]
        s = torch.sigmoid(z)
        return z, s, z * s

    y, ey = torch.zeros(2, B, T, dim, dtype=torch.float64)
    before, M, E = [], h.abs(), torch.zeros_like(h)
    for t in range(T):
        before.append((h, M, E))
        h, M, E = token(p, t, h, M, E)
        out, err = h, E
        if width == 3 * dim:
            _, _, zs = gate_of(p, t)
            out, err = h * zs, (E + 2.0**-19 * h.abs()) * zs.abs()
        y[:, t], ey[:, t] = torch.where(t < n, out, 0.0), torch.where(t < n, err, 0.0)
    last = h, E
    if keep == "int8":
        for t in range(T):
            if t % EVERY:
                before[t] = token(q, t - 1, *before[t - 1])
    dp, ep = torch.zeros(2, B, T, width, dtype=torch.float64)
    c, Mc, Ec = dh, dh.abs(), torch.zeros_like(dh)
    for t in range(T - 1, -1, -1):
        if t + 1 == seam:
            c = torch.zeros_like(c)
        x, f, k = gates(q, t)
        hp, Mp, Ep = before[t]
        d, parts, errors = dy[:, t], [], []
        up, eu = d, 0.0 * d
        if width == 3 * dim:
            z, s, zs = gate_of(q, t)
            hn, _, En = token(q, t, hp, Mp, Ep)
            slope = s + zs * (1 - s)
            off = 2.0**-18 * (s + (zs * (1 - s)).abs()) + 2.0**-23 * zs.abs()
            parts, errors = [d * hn * slope], [d.abs() * (En * slope.abs() + hn.abs() * off)]
            up, eu = d * zs, 2.0**-19 * (d * zs).abs()
        g, M, E = up + c, up.abs() + Mc, eu + Ec + U * (up.abs() + Mc)
        least = GATE * torch.minimum(f, k)
        errors = [
            k * E + (least + U * k) * M,
            k * f * (E * (hp - x).abs() + M * Ep + M * 2 * GATE * (hp - x).abs() + U * M * (hp.abs() + x.abs())),
        ] + errors
        parts = [g * k, g * (hp - x) * f * k] + parts
        live = t < n
        dp[:, t], ep[:, t] = torch.where(live, torch.cat(parts, -1), 0.0), torch.where(live, torch.cat(errors, -1), 0.0)
        c, Mc, Ec = (torch.where(live, a, b) for a, b in ((g * f, c), (M * f, Mc), (f * E + (least + U * f) * M, Ec)))
    return (y, ey), last, (dp, ep), (c, Ec)


def outside(got, bound):
    """How far beyond its bound and its rounding an element is, at most (0: none is)."""
    want, error = bound
    got = got.detach().cpu()
    allowed = torch.finfo(got.dtype).eps / 2 * want.abs() + error
    allowed = 1.01 * allowed + (2.0**-25 if got.dtype == torch.float16 else 1e-37)
    assert got.isfinite().all()
    return float(((got.double() - want).abs() - allowed).clamp_min(0).max()) if got.numel() else 0.0


def check_bounds(p, D, h0, lengths, dy, dh, keep):
    p, h = p.detach().requires_grad_(), h0.detach().requires_grad_()
    y, last = gated_scan(p, D, h, lengths, keep=keep)
    dp, dh0 = torch.autograd.grad((y, last), (p, h), (dy, dh))
    for what, got, bound in zip(("y", "h_last", "dp", "dh0"), (y, last, dp, dh0), bounded(p, D, h0, lengths, dy, dh, keep)):
        assert outside(got, bound) == 0, (what, outside(got, bound))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("keep", ["input", "int8"])
@pytest.mark.parametrize("gate", [True, False], ids=["gate", "plain"])
@pytest.mark.parametrize("B,T,D", [(3, 1, 5), (3, 37, 33), (2, 150, 40)])
def test_every_element_is_within_its_bound(device, dtype, keep, gate, B, T, D):
    p, h0, dy, dh = inputs(B, T, D, dtype, device, gate)
    lengths = torch.tensor([T, T // 2, 1][:B], device=device)
    check_bounds(p, D, h0, lengths, dy, dh, keep)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("keep", ["input", "int8"])
@pytest.mark.parametrize(
    "B,T,D",
    [
        (1, 513, 64),    # chained blocks
        (1, 2049, 40),
        (2, 5000, 33),   # several links
        (4, 2300, 200),  # links of 16 tiles
        (5, 1100, 130),
        (700, 150, 50),  # a block walks several tiles
        (2200, 70, 62),  # a wave walks alone
        (4100, 40, 25),  # staged
        (2100, 40, 100),
        (3, 4, 130),     # short tiles
    ],
)
def test_every_element_of_every_layout(B, T, D, dtype, keep):
    p, h0, dy, dh = inputs(B, T, D, dtype, "cuda")
    lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(2)).cuda()
    lengths[-1] = T
    check_bounds(p, D, h0, lengths, dy, dh, keep)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,T,D", [(1, 513, 64), (2, 2500, 33)])
def test_the_bounds_tell_mistakes(dtype, B, T, D):
    """Planted in the oracle: a carry that is lost at one token, and results 1% too large."""
    p, h0, dy, dh = inputs(B, T, D, dtype, "cpu")
    right = bounded(p, D, h0, None, dy, dh)
    assert all(outside(v.to(dtype if i in (0, 2) else torch.float32), right[i]) == 0 for i, (v, _) in enumerate(right))
    lost = bounded(p, D, h0, None, dy, dh, seam=T // 2)
    for part in range(3):
        at = slice(part * D, (part + 1) * D)
        v, e = right[2][0][..., at], right[2][1][..., at]
        assert outside((v * 1.01).to(dtype), (v, e)) > 0
        if part < 2:  # dz does not know the carry
            assert outside(lost[2][0][..., at].to(dtype), (v, e)) > 0
    assert outside((right[0][0] * 1.01).to(dtype), right[0]) > 0
    assert outside((right[3][0] * 1.01).float(), right[3]) > 0
    first = bounded(p, D, h0, None, dy, dh, seam=1)
    assert outside(first[3][0].float(), right[3]) > 0


@pytest.mark.gpu
def test_more_than_a_launch_takes_is_refused():
    """2^32 threads and more: said before anything is launched."""
    row = torch.zeros(2, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="out of range"):
        gated_scan(row.expand(1, 2**30, 2), 1)
    with pytest.raises(RuntimeError, match="out of range"):
        gated_step(row.expand(2**26, 2), torch.zeros(2**26, 1, device="cuda"))
    y = gated_step(row.expand(2**20, 2), torch.ones(2**20, 1, device="cuda"))
    assert (y == 0.5).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("keep", ["input", "int8"])
@pytest.mark.parametrize("B,T,D", [(3, 4, 20), (2, 90, 33), (2, 100, 130), (1, 1300, 64)])
def test_every_element_with_gates_of_every_size(device, dtype, keep, B, T, D):
    """Tokens that let all of the state go among ones that hold all of it."""
    p, h0, dy, dh = inputs(B, T, D, dtype, "cpu")
    r = (torch.randn(B, T, D, generator=torch.Generator().manual_seed(6)) * 6).clamp(-15.9, 15.9)
    p[..., D : 2 * D] = r.to(dtype)
    lengths = torch.full((B,), T)
    lengths[0] = T - 1
    p, h0, lengths, dy, dh = (t.to(device) for t in (p, h0, lengths, dy, dh))
    check_bounds(p, D, h0, lengths, dy, dh, keep)
