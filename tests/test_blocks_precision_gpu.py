"""What the training-block operators (muzero_amd.blocks) lose to rounding where float32 has few digits to spare, against
float64.  Bounds are derived, not fitted; u = 2^-24 is float32's half step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, t=torch.float32, scale=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(t)


def within(got, ref, bound, what):
    bound = bound + half(got.dtype) * (ref.abs() + bound) + tiny(got.dtype)
    bad = ~((got.double() - ref).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:3].tolist(), ref[bad][:3].tolist(), bound[bad][:3].tolist())


def layer_norm_bounds(x, w, dy, eps):
    """The definition in float64 and the room that float32 needs when the mean's own rounding does not count.

    With d the additions a term of a row's sum passes through, a float32 mean m0 is off by e = (d + 2) u max|x|.  The
    deviations x - m0 are off by u of themselves, their mean t by (d + 3) u of their mean size, and so what is left,
    x - m0 - t, by E = (d + 6) u (|dev| + mean|dev| + e) in all: of e only its product with u stays.  The variance is
    off by (d + 6) u (var + 2 e^2)."""
    c = x.shape[1]
    d = 24 + max(16, c / 1024)
    xd, dyd, wd = x.double(), dy.double(), w.double()
    dev = xd - xd.mean(1, keepdim=True)
    var = (dev ** 2).mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    xh = dev * rstd
    e = (d + 2) * U * xd.abs().amax(1, keepdim=True)
    e_dev = (d + 6) * U * (dev.abs() + dev.abs().mean(1, keepdim=True) + e)
    rel = (d + 6) * U * (var + 2 * e ** 2) / (var + eps) + 4 * U
    e_xh = rstd * e_dev + xh.abs() * rel
    g = dyd * wd
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    size = rstd * (dev.abs() + e)                        # what the sums of dx are made of
    e_m1 = (d + 2) * U * g.abs().mean(1, keepdim=True)
    e_m2 = (d + 8) * U * ((g.abs() * size).mean(1, keepdim=True) + rstd * e * m1.abs() + rstd * e * g.abs().mean(1, keepdim=True))
    e_m2 = e_m2 + (g.abs() * e_xh).mean(1, keepdim=True)
    inner = g.abs() + m1.abs() + (xh * m2).abs()
    e_dx = rstd * (e_m1 + xh.abs() * e_m2 + e_xh * (m2.abs() + e_m2) + 6 * U * inner) + rel * rstd * inner
    dc = x.shape[0] + 70
    dw, e_dw = (dyd * xh).sum(0), (dc * U * (dyd * xh).abs() + dyd.abs() * e_xh * (1 + dc * U)).sum(0)
    return xh, e_xh, rstd * (g - m1 - xh * m2), e_dx, dw, e_dw, dyd.sum(0), dc * U * dyd.abs().sum(0)


def check_layer_norm(x, w, b, dy, eps=1e-5):
    from muzero_amd import blocks
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    y = blocks.layer_norm(*leaves, eps=eps)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    xh, e_xh, dxr, e_dx, dwr, e_dw, dbr, e_db = layer_norm_bounds(x, w, dy, eps)
    wd, bd = w.double(), b.double()
    within(y.detach(), xh * wd + bd, e_xh * wd.abs() + 3 * U * (xh * wd).abs() + 2 * U * bd.abs(), "y")
    within(dx, dxr, e_dx, "dx")
    within(dw, dwr, e_dw, "dweight")
    within(db, dbr, e_db, "dbias")
    only = torch.autograd.grad(blocks.layer_norm(x, leaves[1], b, eps=eps), leaves[1], dy)[0]       # without dx: the same bits
    assert torch.equal(only, dw)


@pytest.mark.parametrize("c", [24, 100, 257, 777, 1001, 3000, 8191, 16001, 20001, 40000])
def test_constant_rows_give_the_bias(c):
    """Values that are no short binary fractions at widths that are no powers of two: nothing of the mean's rounding may
    be left in y."""
    g = gen(c)
    values = torch.tensor([12345.6, 54321.0, 1000.1, 100.1, -7.3e6, 0.1, -3.3e-5], device="cuda")
    x = values[:, None].expand(7, c).contiguous()
    check_layer_norm(x, normal(g, c, mean=1.0), normal(g, c), normal(g, 7, c))


@pytest.mark.parametrize("offset", [1e2, 1e4, 1e6])
@pytest.mark.parametrize("rows,c", [(6, 40), (40, 777), (300, 1001), (5, 9000), (4, 20001)])
def test_common_offset_costs_no_digits(rows, c, offset):
    g = gen(rows + c)
    x = normal(g, rows, c, mean=offset)
    check_layer_norm(x, normal(g, c, mean=1.0), normal(g, c), normal(g, rows, c))


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("c", [100, 1001, 5000, 20001])
def test_common_offset_in_16_bits(c, t):
    g = gen(c + 1)
    x = torch.cat([normal(g, 20, c, t=TYPES[t], mean=100.0), torch.full((2, c), 1000.1, device="cuda").to(TYPES[t])])
    check_layer_norm(x, normal(g, c, mean=1.0), normal(g, c), normal(g, 22, c, t=TYPES[t]))


def test_rows_whose_squares_overflow_and_bad_rows():
    """Deviations of 1e30 have no float32 square: y is the bias, as before and as in torch; NaN and infinity stay in their row."""
    from muzero_amd import blocks
    g = gen(5)
    for c in (100, 3000, 20001):
        x, b = normal(g, 4, c), normal(g, c)
        good = blocks.layer_norm(x, None, b)
        x[1] *= 1e30
        x[2, 5] = float("nan")
        x[3, c - 1] = float("inf")
        y = blocks.layer_norm(x, None, b)
        assert torch.equal(y[0], good[0]) and torch.equal(y[1], b) and torch.isnan(y[2]).all() and torch.isnan(y[3]).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,c", [(9000, 7), (5000, 300), (3000, 1001), (1500, 4096), (1500, 4097), (700, 9001), (600, 16384),
                                    (700, 20001), (300, 65537), (3, 70000)])
def test_layer_norm_stays_inside_its_workspace(rows, c, t):
    """The workspace asked for between canaries and full of NaN, dx wanted and not: the bits of the Python entry point."""
    from muzero_amd import _lib, blocks
    from tests.test_blocks_gpu import Canary
    g, t = gen(rows + c), TYPES[t]
    x, dy = normal(g, rows, c, t=t), normal(g, rows, c, t=t)
    w, b = normal(g, c, mean=1.0).requires_grad_(), normal(g, c).requires_grad_()
    leaf = x.detach().requires_grad_()
    dx, dw, db = torch.autograd.grad(blocks.layer_norm(leaf, w, b), (leaf, w, b), dy)
    p, s = (lambda v: v.data_ptr()), _lib.current_stream()
    dt = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[t]
    need = _lib.lib().mz_layer_norm_workspace_bytes(rows, c)
    for with_dx in (True, False):
        y, stats, ws = Canary(rows * c, t), Canary(2 * rows, torch.float32), Canary(need // 4, torch.float32)
        out = [Canary(rows * c, t), Canary(c, torch.float32), Canary(c, torch.float32)]
        _lib.call("mz_layer_norm_fwd", p(x), c, p(w), p(b), 0, 1e-5, rows, c, dt, y.ptr(), stats.ptr(), stats.ptr() + 4 * rows, s)
        _lib.call("mz_layer_norm_bwd", p(x), c, p(dy), c, p(w), 0, stats.ptr(), stats.ptr() + 4 * rows, rows, c, dt,
                  out[0].ptr() if with_dx else None, out[1].ptr(), out[2].ptr(), ws.ptr(), need, s)
        assert (ws.all[:512] == 7.0).all() and (ws.all[-512:] == 7.0).all()
        for canary, want in zip(out[1 - with_dx:], (dx, dw, db)[1 - with_dx:]):
            canary.check("layer_norm")
            assert torch.equal(canary.inner, want.reshape(-1))


# ------------------------------------------------------------------------------------------- gated feed-forward
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [9, 64, 300])
def test_gated_ff_long_sums_beside_large_biases(rows, t):
    """2^20 terms of 1.9 x 2^-18 beside a bias of 4096: 32 of them are below the last float32 digit of the bias, all of them two
    steps of a float16 result.  Gradients: dW_up = sum act(g), which takes g's value, and dW_gate = sum dh u."""
    from muzero_amd import blocks
    t = TYPES[t]
    k, f = 1 << 20, 24
    x = torch.ones(rows, k, dtype=t, device="cuda")
    wg = torch.full((f, k), 1.9 * 2.0 ** -18, device="cuda").to(t)
    wu, bg, bu = torch.zeros_like(wg), torch.full((f,), 4096.0, dtype=t, device="cuda"), torch.ones(f, dtype=t, device="cuda")
    leaves = [v.requires_grad_() for v in (wg, wu)]
    h = blocks.gated_ff(x, *leaves, bg, bu, activation="relu")
    gate = 4096.0 + k * wg[0, 0].double().item()
    # the sum's own error: K / 16 additions at most (float32: K) that each lose u of at most its 8 - 2^20 u 8 = 0.5
    n = k if t == torch.float32 else k // 16
    room = torch.full((rows, f), n * U * (gate - 4096.0) + 3 * U * gate, dtype=torch.float64, device="cuda")
    within(h.detach(), torch.full_like(room, gate), room, "h")
    dh = torch.full((rows, f), 2.0 ** -10, dtype=t, device="cuda")
    dwg, dwu = torch.autograd.grad(h, leaves, dh)
    # every term is the same: one rounding of dg = 2^-10 (exact) and of du = 2^-10 gate, which is held in t, and the sum's
    step = half(t) if t != torch.float32 else 0.0
    ref, off = rows * 2.0 ** -10 * gate, rows * 2.0 ** -10 * (room[0, 0].item() + step * gate)
    bound = torch.full((f, k), off + (rows + 40) * U * ref, dtype=torch.float64, device="cuda")
    within(dwu, torch.full_like(bound, ref), bound, "dw_up")
    assert (dwg == rows * 2.0 ** -10).all()


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("rows,k,f,carried", [(32, 256, 256, True), (90, 130, 72, True), (8, 2048, 1024, True), (1, 1500, 8192, False),
                                              (2, 4100, 4000, False), (33, 256, 256, False), (130, 200, 1000, False),
                                              (2500, 512, 700, False)])
def test_gated_ff_gradients_are_off_by_one_rounding_or_two(rows, k, f, carried, t):
    """The documented error of 16-bit gradients, on both sides of both limits.  Rounding a number m 2^e, 1 <= m < 2, is off by a
    uniform error of up to half = 2^(e - p): RMS half / (sqrt(3) m) relative, and with m spread over its logarithm, E 1/m^2 =
    3 / (8 ln 2), sqrt(3 / (8 ln 2) / 3) half = 0.425 half.  Terms that were rounded before give the sum as much again,
    independent of the result's: sqrt(2) of it.  A tenth of room: at 10^4 elements and more the RMS itself is sharp to a
    hundredth, the spread of m is not exactly that."""
    from muzero_amd import blocks
    t = TYPES[t]
    g = gen(rows + f)
    x, wg, wu = (normal(g, *s, t=t, scale=sc).requires_grad_() for s, sc in (((rows, k), 1.0), ((f, k), k ** -0.5), ((f, k), k ** -0.5)))
    dh = normal(g, rows, f, t=t)
    got = torch.autograd.grad(blocks.gated_ff(x, wg, wu), (x, wg, wu), dh)
    xd, gd, ud = (v.detach().double() for v in (x, wg, wu))
    gate, up = xd @ gd.t(), xd @ ud.t()
    sig = torch.sigmoid(gate)
    dg, du = dh.double() * up * sig * (1 + gate * (1 - sig)), dh.double() * gate * sig
    one = (3 / (8 * math.log(2)) / 3) ** 0.5 * half(t)
    for v, ref, name in zip(got, (dg @ gd + du @ ud, dg.t() @ xd, du.t() @ xd), ("x", "w_gate", "w_up")):
        off = ((v.double() - ref).norm() / ref.norm()).item()
        if v.numel() >= 10000:
            assert off <= 1.1 * one * (1 if carried else 2 ** 0.5), (name, off, one)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid"])
def test_gated_ff_activations_keep_their_digits_far_from_zero(activation, rows, t):
    """Gates that are given exactly (one column of ones): activation and slope relative to their own size, however small.
    Room: an exponential of g is off by u |g|, as g log2(e) is rounded.  Of g^2 / 2: erfc takes z = g sqrt(1/2), off by u for the
    constant and u for the product, so z^2 = g^2 / 2 by 4 u, and its exponential by 4 u times that.  24 u for the functions
    and products themselves; 16-bit types the hardware's exponential, 4 u of its argument more."""
    from muzero_amd import blocks
    t = TYPES[t]
    reach = {"silu": 80.0, "sigmoid": 80.0, "gelu": 12.0}[activation]
    if t == torch.float16:                           # results in float16's normal range
        reach = {"silu": 10.0, "sigmoid": 9.0, "gelu": 3.8}[activation]
    gate = torch.linspace(-reach, reach, 1001, device="cuda").to(t)
    f = gate.numel()
    x = torch.ones(rows, 1, dtype=t, device="cuda")
    wg, wu = gate[:, None].clone().requires_grad_(), torch.ones(f, 1, dtype=t, device="cuda").requires_grad_()
    h = blocks.gated_ff(x, wg, wu, activation=activation)
    dh = torch.zeros(rows, f, dtype=t, device="cuda")
    dh[1] = 1.0
    dwg, dwu = torch.autograd.grad(h, (wg, wu), dh)     # one row: act'(g) and act(g) themselves
    g = gate.double()
    sig, small = torch.sigmoid(g), torch.sigmoid(-g)
    cdf = 0.5 * torch.special.erfc(-g * 0.5 ** 0.5)
    density = torch.exp(-0.5 * g * g) / (2 * math.pi) ** 0.5
    act, slope, size = {"silu": (g * sig, sig * (1 + g * small), sig * (1 + g.abs() * small)), "sigmoid": (sig, sig * small, sig * small),
                        "gelu": (g * cdf, cdf + g * density, cdf + g.abs() * density)}[activation]
    power = g * g / 2 if activation == "gelu" else g.abs()
    rel = (24 + (4 if activation == "gelu" else 2) * power + (0 if t == torch.float32 else 4 * power)) * U
    within(h.detach(), act.expand(rows, f), (rel * act.abs()).expand(rows, f), "h")
    # rounded to the type on the way, 3 rows with the remainder carried, 40 without
    again = 0.0 if t == torch.float32 else half(t) if rows * f > 8192 else half(t) ** 2
    within(dwu[:, 0], act, (rel + again) * act.abs() + tiny(t), "dw_up")
    within(dwg[:, 0], slope, rel * size + again * slope.abs() + tiny(t), "dw_gate")
