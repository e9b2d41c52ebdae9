"""Residual-block operators (favae_hip/blocks.py) against plain fp64 formulas: group norm with an activation, matrix product with bias,
activation and residual, their gradients, and 8-bit activation checkpoints.

Bounds.  u = 2^-24 (half a step of fp32).  A stored value is off by half a step of its type.  Sums inside the kernels are trees over
runs of at most a few hundred terms, so that a sum of t terms is off by at most SUM * u * sum|term| with SUM = 400 + (t's share of one
lane, stated where it is larger); matrix products accumulate K terms in one chain: (K + 8) u sum|x w|.  The activations have slope at
most 1.13 and curvature at most 1.2; their exp and reciprocal add (|z| + 8) 4 u of relative error."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
SUM = 400 * U
F32, BF16, F64 = torch.float32, torch.bfloat16, torch.float64
ACTS = ["none", "lrelu", "silu", "gelu_tanh"]
SLOPE, CURVE = 1.13, 1.2


def B():
    from favae_hip import blocks
    return blocks


def half(t):
    return torch.finfo(t).eps / 2


def act64(z, act):
    if act == "none":
        return z, torch.ones_like(z)
    if act == "lrelu":
        return torch.where(z > 0, z, 0.01 * z), torch.where(z > 0, 1.0, 0.01).to(z)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    c = math.sqrt(8 / math.pi)
    s = torch.sigmoid(c * (z + 0.044715 * z ** 3))
    return z * s, s * (1 + z * (1 - s) * c * (1 + 0.134145 * z * z))


def close(got, want, bound, dtype=None):
    """|got - want| <= half a step of the stored type + bound, everywhere."""
    assert got.shape == want.shape
    lim = bound + half(dtype or got.dtype) * (want.abs() + bound) + 1e-37
    bad = (got.double() - want).abs() - lim
    assert not torch.isnan(got).any()
    assert bad.numel() == 0 or bad.max() <= 0, (bad.max().item(), (got.double() - want).abs().max().item())


def rnd(gen, *shape, dtype=F32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale + shift).to(dtype)


def gen(*key):
    return torch.Generator(device=DEV).manual_seed(hash(tuple(int(k) for k in key)) % (1 << 31))


# ---- 8-bit activations ---------------------------------------------------------------------------------------------------
def ref_pack(x):
    """The format from its definition, block by block, in fp64 on the host."""
    x = x.double().cpu()
    R, C = x.shape
    nb = (C + 31) // 32
    q, e = torch.zeros(R, C, dtype=torch.int8), torch.zeros(R, nb, dtype=torch.uint8)
    for b in range(nb):
        blk = x[:, 32 * b:32 * b + 32]
        for r in range(R):
            v = blk[r]
            if not torch.isfinite(v).all():
                e[r, b] = 255
                continue
            k = -126
            while k < 121 and torch.round(v.abs().max() * 2.0 ** -k) > 127:
                k += 1
            q[r, 32 * b:32 * b + 32] = torch.round(v * 2.0 ** -k).clamp(-127, 127).to(torch.int8)
            e[r, b] = k + 127
    return q, e


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("R,C", [(1, 1), (3, 31), (5, 32), (2, 33), (7, 40), (4, 64), (3, 129), (33, 8), (2, 1024)])
def test_ckpt8_is_the_format_bit_for_bit(R, C, dtype):
    b = B()
    x = rnd(gen(R, C), R, C, dtype=dtype) * torch.exp2(torch.randint(-40, 40, (R, 1), generator=gen(C, R), device=DEV).float()).to(dtype)
    x[0, :min(C, 32)] = 0                                   # a block of zeros
    ck = b.ckpt8_pack(x)
    q, e = ref_pack(x)
    assert torch.equal(ck.q.cpu(), q) and torch.equal(ck.e.cpu(), e)
    want = q.double() * torch.exp2(e.double() - 127).repeat_interleave(32, 1)[:, :C]
    for t in (F32, BF16):
        assert torch.equal(b.ckpt8_unpack(ck, t).cpu().double(), want)      # decoded values are exact in both types
    # no value is further than half a step of its block from what was packed, nor a step above 2^-6 of the block's largest
    step = torch.exp2(e.double() - 127).repeat_interleave(32, 1)[:, :C]
    assert ((want - x.double().cpu()).abs() <= 0.5 * step).all()


def test_ckpt8_extremes_and_faults():
    b = B()
    big, tiny = torch.finfo(F32).max, 2.0 ** -149
    x = torch.zeros(8, 64, device=DEV)
    x[0, 3], x[0, 5] = big, -big
    x[1, 0] = tiny
    x[2, 0], x[2, 1] = 2.0 ** -126, 2.0 ** -127
    x[3, 7] = float("inf")
    x[4, 40] = float("nan")
    x[5, 0], x[5, 1] = 127.5, 1.0                           # rounds to 128 steps of 1: the step is 2
    x[6, 0], x[6, 1], x[6, 2] = 127.0, 0.5, 1.5             # ties to even: 0 and 2
    x[7, 0] = -float("inf")
    ck = b.ckpt8_pack(x)
    q, e = ref_pack(x)
    assert torch.equal(ck.q.cpu(), q) and torch.equal(ck.e.cpu(), e)
    v = b.ckpt8_unpack(ck)
    assert torch.isnan(v[3, :32]).all() and (v[3, 32:] == 0).all() and torch.isnan(v[4, 32:]).all() and torch.isnan(v[7, :32]).all()
    assert torch.isfinite(v[0]).all() and v[0, 3] == 127 * 2.0 ** 121 and v[5, 0] == 128 and v[6, 1] == 0 and v[6, 2] == 2
    assert torch.isfinite(b.ckpt8_unpack(ck, BF16)[0]).all()


def test_ckpt8_strides_and_empty():
    b = B()
    wide = rnd(gen(1), 9, 100)
    for x in (wide[:, 3:67], wide[:, 4:36], wide[::2, 8:72], wide.to(BF16)[:, 1:34], wide.view(3, 3, 100)[:, :, :64]):
        ck, ref = b.ckpt8_pack(x), b.ckpt8_pack(x.contiguous())
        assert torch.equal(ck.q, ref.q) and torch.equal(ck.e, ref.e)
        out = torch.full(x.shape[:-1] + (x.shape[-1] + 5,), 7.0, device=DEV, dtype=x.dtype)
        b.ckpt8_unpack(ck, out=out[..., 2:-3])
        assert torch.equal(out[..., 2:-3], b.ckpt8_unpack(ref)) and (out[..., :2] == 7).all() and (out[..., -3:] == 7).all()
    for shape in ((0, 8), (4, 0), (0,)):
        x = torch.empty(shape, device=DEV)
        assert b.ckpt8_unpack(b.ckpt8_pack(x)).shape == x.shape


# ---- group norm ----------------------------------------------------------------------------------------------------------
GN = [(1, 1, 1, 1), (2, 1, 8, 2), (3, 7, 10, 5), (1, 4, 1024, 32), (3, 64, 64, 8), (2, 4096, 64, 16), (5, 195, 210, 30), (700, 1, 64, 8),
      (3, 2, 24, 24), (2, 9000, 16, 2), (1, 70000, 8, 1), (2, 5, 8192, 1), (1, 3, 4099, 1), (2, 300, 2050, 2), (4, 33, 33, 3), (130, 16, 256, 4)]


def gn_ref(x, gamma, beta, G, act, eps=1e-5):
    """y, mean, rstd in fp64, the bound of z's error, and z and xh."""
    n, c = x.shape[0], x.shape[-1]
    xg = x.double().reshape(n, -1, G, c // G)
    mean = xg.mean((1, 3))
    var = (xg - mean[:, None, :, None]).square().mean((1, 3))
    rstd = (var + eps).rsqrt()
    xh = ((xg - mean[:, None, :, None]) * rstd[:, None, :, None]).reshape(n, -1, c)
    z = xh * gamma.double() + beta.double()
    mean_err = SUM * xg.abs().mean((1, 3)) + U * mean.abs()
    # the squared distances: relative SUM, and twice the mean's rounding against the spread
    rstd_rel = SUM + 4 * U + mean_err.square() * rstd.square()
    xh_err = (mean_err * rstd)[:, None, :, None].expand(xg.shape).reshape(n, -1, c) + xh.abs() * (rstd_rel[:, None, :, None].expand(xg.shape).reshape(n, -1, c) + 2 * U)
    z_err = gamma.double().abs() * xh_err + 4 * U * (z.abs() + beta.double().abs())
    return act64(z, act)[0], mean, rstd, z, z_err, mean_err, rstd_rel


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,S,C,G", GN)
def test_group_norm_act(N, S, C, G, dtype):
    b = B()
    g = gen(N, S, C, G)
    x = rnd(g, N, S, C, dtype=dtype, scale=1.7, shift=3.0)
    gamma, beta = rnd(g, C, scale=0.3, shift=1.0), rnd(g, C, scale=0.5)
    for act in ACTS:
        y, mean, rstd = b.group_norm_act(x, G, gamma, beta, act=act)
        want, m, r, z, z_err, m_err, r_rel = gn_ref(x, gamma, beta, G, act)
        close(mean, m, m_err)
        close(rstd, r, r * r_rel)
        close(y, want, SLOPE * z_err + (z.abs() + 8) * 4 * U * want.abs())
        assert y.dtype == dtype and mean.dtype == rstd.dtype == F32


def gn_bwd_check(b, N, S, C, G, dtype, act, ck, g):
    x = rnd(g, N, S, C, dtype=dtype, scale=1.7, shift=3.0)
    dy = rnd(g, N, S, C, dtype=dtype)
    gamma, beta = rnd(g, C, scale=0.3, shift=1.0), rnd(g, C, scale=0.5)
    _, mean, rstd = b.group_norm_act(x, G, gamma, beta, act=act)
    src = b.ckpt8_pack(x) if ck else x
    xv = b.ckpt8_unpack(src, F32) if ck else x
    dx, dg, db = b.group_norm_act_bwd(dy, src, G, gamma, beta, mean, rstd, act=act)
    rep = lambda t: t.double().repeat_interleave(C // G, 1)[:, None, :]
    ga, be = gamma.double(), beta.double()
    d = xv.double() - rep(mean)
    xh = d * rep(rstd)
    xh_err = 2 * U * xh.abs()
    z = xh * ga + be
    z_err = ga.abs() * xh_err + 2 * U * (z.abs() + be.abs())
    _, slope = act64(z, act)
    dz = dy.double() * slope
    dz_err = dy.double().abs() * (CURVE * z_err + (z.abs() + 8) * 4 * U) if act != "none" else torch.zeros_like(dz)
    if act == "lrelu":                                       # within the rounding of z the kink may fall on either side
        dz_err = dz_err + torch.where(z.abs() <= z_err, 0.99 * dy.double().abs(), 0.0)
    close(db, dz.sum((0, 1)), dz_err.sum((0, 1)) + SUM * dz.abs().sum((0, 1)))
    close(dg, (dz * xh).sum((0, 1)), (dz_err * xh.abs() + dz.abs() * xh_err).sum((0, 1)) + SUM * (dz * xh).abs().sum((0, 1)))
    grp = lambda t: t.sum(1).reshape(N, G, C // G).sum(2)
    m = S * (C // G)
    s1, s2 = grp(ga * dz), grp(ga * dz * xh)
    s1_err = grp(ga.abs() * dz_err) + SUM * grp((ga * dz).abs())
    s2_err = grp(ga.abs() * (dz_err * xh.abs() + dz.abs() * xh_err)) + SUM * grp((ga * dz * xh).abs())
    want = rep(rstd) * (ga * dz - (rep(s1) + xh * rep(s2)) / m)
    size = rep(rstd) * ((ga * dz).abs() + (rep(s1).abs() + (xh * rep(s2)).abs()) / m)
    err = rep(rstd) * (ga.abs() * dz_err + (rep(s1_err) + xh.abs() * rep(s2_err) + xh_err * rep(s2).abs()) / m) + 6 * U * size
    close(dx, want, err)
    assert dx.dtype == dtype and dg.dtype == db.dtype == F32


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,S,C,G", GN)
def test_group_norm_act_bwd(N, S, C, G, dtype):
    for act in ACTS:
        for ck in (False, True):
            gn_bwd_check(B(), N, S, C, G, dtype, act, ck, gen(N, S, C, G, ck))


# channel counts off the vector grid: blocks of groups with a short last one, several of one sample's blocks, small workgroups, several samples in
# one, rows narrower than a vector, chunks
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,S,C,G", [(2, 4000, 945, 945), (300, 50, 231, 33), (100, 700, 165, 5), (64, 1023, 99, 33), (500, 9, 66, 2), (40, 12, 7, 7),
                                     (600, 3, 5, 1), (3, 20, 20, 4), (1, 20000, 33, 3), (260, 64, 1023, 31)])
def test_group_norm_odd_channels(N, S, C, G, dtype):
    b = B()
    g = gen(N, S, C, G, 1)
    x = rnd(g, N, S, C, dtype=dtype, scale=1.7, shift=3.0)
    gamma, beta = rnd(g, C, scale=0.3, shift=1.0), rnd(g, C, scale=0.5)
    y, mean, rstd = b.group_norm_act(x, G, gamma, beta, act="silu")
    want, m, r, z, z_err, m_err, r_rel = gn_ref(x, gamma, beta, G, "silu")
    close(mean, m, m_err)
    close(rstd, r, r * r_rel)
    close(y, want, SLOPE * z_err + (z.abs() + 8) * 4 * U * want.abs())
    xi = x.clone()
    assert torch.equal(b.group_norm_act(xi, G, gamma, beta, act="silu", out=xi)[0], y)           # in place
    dy = rnd(g, N, S, C, dtype=dtype)
    dx = b.group_norm_act_bwd(dy, x, G, gamma, beta, mean, rstd, act="silu")[0]
    di = dy.clone()
    assert torch.equal(b.group_norm_act_bwd(di, x, G, gamma, beta, mean, rstd, act="silu", out=di)[0], dx)
    for ck in (False, True):
        gn_bwd_check(b, N, S, C, G, dtype, "silu", ck, gen(N, S, C, G, 2 + ck))


@pytest.mark.parametrize("N,S,C,G", [(3, 50, 210, 30), (300, 50, 231, 33), (2, 2000, 99, 33), (1, 30000, 33, 11)])
def test_group_norm_nan_stays_in_its_group_with_odd_channels(N, S, C, G):
    b = B()
    g = gen(N, S, C, G, 9)
    x, dy = rnd(g, N, S, C, dtype=BF16), rnd(g, N, S, C, dtype=BF16)
    gamma, beta = torch.ones(C, device=DEV), torch.zeros(C, device=DEV)
    cg = C // G
    bad = torch.zeros(N, S, C, dtype=torch.bool, device=DEV)
    for grp in (0, G // 2, G - 1):
        x[N - 1, S - 1, grp * cg + cg - 1] = float("nan")
        bad[N - 1, :, grp * cg:(grp + 1) * cg] = True
    y, m, r = b.group_norm_act(x, G, gamma, beta, act="silu")
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
    dx, dg, db = b.group_norm_act_bwd(dy, x, G, gamma, beta, m, r, act="silu")
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()
    cols = bad.flatten(0, 1).any(0)
    assert torch.isnan(dg[cols]).all() and torch.isfinite(dg[~cols]).all() and torch.isnan(db[cols]).all() and torch.isfinite(db[~cols]).all()


def test_group_norm_gradients_against_differences():
    """dx, dgamma, dbeta of the kernels against central differences of the fp64 forward formula along random directions."""
    b = B()
    g = gen(42)
    N, S, C, G = 2, 12, 24, 4
    x, dy = rnd(g, N, S, C), rnd(g, N, S, C)
    gamma, beta = rnd(g, C, scale=0.3, shift=1.0), rnd(g, C, scale=0.5)
    for act in ("none", "silu", "gelu_tanh"):
        _, mean, rstd = b.group_norm_act(x, G, gamma, beta, act=act)
        grads = b.group_norm_act_bwd(dy, x, G, gamma, beta, mean, rstd, act=act)
        f = lambda t: (gn_ref(t[0], t[1], t[2], G, act)[0] * dy.double()).sum()
        args = [x.double(), gamma.double(), beta.double()]
        for k in range(3):
            v = torch.randn(args[k].shape, generator=g, device=DEV, dtype=F64)
            up, dn = list(args), list(args)
            h = 1e-5
            up[k], dn[k] = args[k] + h * v, args[k] - h * v
            diff = (f(up) - f(dn)) / (2 * h)
            # third derivative times h^2 is below 1e-8; the kernels' fp32 sums: SUM of the absolute terms
            assert abs((grads[k].double() * v).sum() - diff) <= 1e-7 * (grads[k].double() * v).abs().sum() + SUM * (dy.double().abs().sum() * v.abs().max())


def test_group_norm_layouts_in_place_and_empty():
    b = B()
    g = gen(7)
    big = rnd(g, 3, 10, 12, 48, dtype=BF16)
    gamma, beta = rnd(g, 32), rnd(g, 32)
    for x in (big[:, :, :, :32], big[:, :, :, 5:37], big[:, 2:3, :, 8:40], big[1:2, :, :, 16:48]):
        dy = rnd(g, *x.shape, dtype=BF16)
        y, m, r = b.group_norm_act(x, 4, gamma, beta, act="silu")
        y2, m2, r2 = b.group_norm_act(x.contiguous(), 4, gamma, beta, act="silu")
        close(y, y2.double(), half(BF16) * y2.double().abs())        # another vector width sums in another order
        out = torch.full(x.shape[:-1] + (40,), 9.0, dtype=BF16, device=DEV)
        b.group_norm_act(x, 4, gamma, beta, act="silu", out=out[..., 4:36])
        assert torch.equal(out[..., 4:36], y) or (out[..., 4:36].float() - y.float()).abs().max() <= 2 ** -7 * y.float().abs().max()
        assert (out[..., :4] == 9).all() and (out[..., 36:] == 9).all()
        dx = b.group_norm_act_bwd(dy, x, 4, gamma, beta, m, r, act="silu")[0]
        dx2 = b.group_norm_act_bwd(dy, x.contiguous(), 4, gamma, beta, m, r, act="silu")[0]
        assert (dx.float() - dx2.float()).abs().max() <= 2 ** -7 * dx2.float().abs().max()
    # a channels_last convolution output is a view of this layout
    nchw = rnd(g, 2, 32, 5, 6).to(memory_format=torch.channels_last)
    y, _, _ = b.group_norm_act(nchw.permute(0, 2, 3, 1), 8, gamma, beta, act="lrelu")
    want = gn_ref(nchw.permute(0, 2, 3, 1).contiguous(), gamma, beta, 8, "lrelu")
    close(y.reshape(2, 30, 32), want[0], SLOPE * want[4] + 8 * U * want[0].abs())
    # in place, forward and backward
    x = rnd(g, 4, 50, 32)
    dy = rnd(g, 4, 50, 32)
    y, m, r = b.group_norm_act(x, 4, gamma, beta, act="gelu_tanh")
    xi, di = x.clone(), dy.clone()
    assert b.group_norm_act(xi, 4, gamma, beta, act="gelu_tanh", out=xi)[0] is xi and torch.equal(xi, y)
    dx = b.group_norm_act_bwd(dy, x, 4, gamma, beta, m, r, act="gelu_tanh")[0]
    assert torch.equal(b.group_norm_act_bwd(di, x, 4, gamma, beta, m, r, act="gelu_tanh", out=di)[0], dx)
    # nothing in, nothing out
    y, m, r = b.group_norm_act(torch.empty(0, 5, 32, device=DEV), 4, gamma, beta)
    assert y.shape == (0, 5, 32) and m.shape == (0, 4)
    e = torch.empty(3, 0, 32, device=DEV)
    y, m, r = b.group_norm_act(e, 4, gamma, beta)
    assert y.shape == e.shape and (m == 0).all() and torch.allclose(r, torch.full_like(r, 1e-5 ** -0.5))
    for t in (e, torch.empty(0, 5, 32, device=DEV)):
        st = torch.zeros(t.shape[0], 4, device=DEV)
        dx, dg, db = b.group_norm_act_bwd(t, t, 4, gamma, beta, st, st)
        assert dx.shape == t.shape and (dg == 0).all() and (db == 0).all()
    for wide in ((0, 5, 4099), (0, 5, 8192)):                 # an empty batch of what would go in chunks
        t, v = torch.empty(wide, device=DEV), torch.ones(wide[-1], device=DEV)
        st = torch.zeros(0, 1, device=DEV)
        assert b.group_norm_act(t, 1, v, v)[0].shape == wide
        dx, dg, db = b.group_norm_act_bwd(t, t, 1, v, v, st, st)
        assert dx.shape == wide and (dg == 0).all() and (db == 0).all()
    # a constant group: variance 0
    y, m, r = b.group_norm_act(torch.full((2, 9, 32), 5.0, device=DEV), 4, gamma, beta)
    assert (m == 5).all() and torch.equal(y, beta.expand(2, 9, 32))


def test_group_norm_far_mean_and_nan_stays_in_its_group():
    b = B()
    g = gen(8)
    x = rnd(g, 2, 500, 32, scale=0.01, shift=1000.0)         # spread 1e-5 of the mean: squares minus square of the mean would be noise
    gamma, beta = torch.ones(32, device=DEV), torch.zeros(32, device=DEV)
    y, m, r = b.group_norm_act(x, 4, gamma, beta, eps=0.0)
    xg = x.double().reshape(2, 500, 4, 8)
    sd = xg.var((1, 3), unbiased=False).sqrt()
    m_err = (SUM + U) * xg.abs().mean((1, 3))
    assert ((r.double() * sd - 1).abs() <= SUM + (m_err / sd) ** 2).all()
    x[0, 3, 9] = float("nan")
    x[1, 4, 0] = float("inf")
    y, m, r = b.group_norm_act(x, 4, gamma, beta)
    bad = torch.zeros(2, 500, 32, dtype=torch.bool, device=DEV)
    bad[0, :, 8:16] = True
    bad[1, :, 0:8] = True
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,S,C,G", [(5, 65, 96, 8), (2, 7, 40, 5), (3, 9000, 32, 2), (64, 1, 64, 4), (2, 33, 128, 1), (4, 16, 512, 32)])
def test_group_norm_forward_checkpoint_is_the_input_packed(N, S, C, G, dtype):
    b = B()
    wide = rnd(gen(3, N, C), N, S + 1, C + 8, dtype=dtype)
    gamma, beta = torch.ones(C, device=DEV), torch.zeros(C, device=DEV)
    for x in (wide[:, :S, :C].contiguous(), wide[:, :S, 8:], wide[:, :S, 1:C + 1]):
        y, m, r, ck = b.group_norm_act(x, G, gamma, beta, act="silu", ckpt=True)
        ref = b.ckpt8_pack(x.contiguous())
        assert torch.equal(ck.q, ref.q) and torch.equal(ck.e, ref.e)
        y2, m2, r2 = b.group_norm_act(x, G, gamma, beta, act="silu")
        assert (y.float() - y2.float()).abs().max() <= 2 ** -7 * y2.float().abs().max() and (m - m2).abs().max() <= 1e-5


# ---- matrix product ------------------------------------------------------------------------------------------------------
LIN = [(1, 1, 1), (1, 4096, 64), (3, 7, 5), (2, 20, 200), (64, 128, 4096), (129, 130, 65), (200, 33, 523), (130, 256, 64), (256, 384, 192), (1000, 8, 16),
       (17, 300, 8), (5, 1000, 1031), (16, 512, 1024), (40, 264, 520)]      # M, N, K


def lin_bound(x, w, bias):
    k = x.shape[-1]
    return (k + 8) * U * (x.double().abs() @ w.double().abs().t()) + 2 * U * bias.double().abs()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", LIN)
def test_linear_act(M, N, K, dtype):
    b = B()
    g = gen(M, N, K)
    x, w = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype, scale=K ** -0.5)
    bias, res = rnd(g, N, scale=0.3), rnd(g, M, N, dtype=dtype)
    for act in ACTS:
        for with_bias, with_res, save in ((True, True, True), (False, False, False), (True, False, False)):
            bb = bias if with_bias else torch.zeros_like(bias)
            got = b.linear_act(x, w, bias if with_bias else None, act=act, residual=res if with_res else None, save_pre=save)
            u = x.double() @ w.double().t() + bb.double()
            u_err = lin_bound(x, w, bb)
            v = act64(u, act)[0]
            err = SLOPE * u_err + (u.abs() + 8) * 4 * U * v.abs()
            if with_res:
                v = v + res.double()
                err = err + U * v.abs()
            if save:
                got, pre = got
                close(pre, u, u_err)
            close(got, v, err)
            assert got.dtype == dtype


def lin_bwd_check(b, M, N, K, dtype, act, ck, g, dw_dtype=None):
    x, w, dy = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype, scale=K ** -0.5), rnd(g, M, N, dtype=dtype)
    pre = rnd(g, M, N, dtype=dtype, scale=2.0)
    xs, ps = (b.ckpt8_pack(x), b.ckpt8_pack(pre)) if ck else (x, pre)
    xv, pv = (b.ckpt8_unpack(xs, F32).double(), b.ckpt8_unpack(ps, F32).double()) if ck else (x.double(), pre.double())
    buf = torch.full((N, K), float("nan"), dtype=dw_dtype, device=DEV) if dw_dtype else None
    dx, dw, db = b.linear_act_bwd(dy, xs, w, act=act, pre=None if act == "none" else ps, dw=buf)
    slope = act64(pv, act)[1]
    du = dy.double() * slope
    du_err = dy.double().abs() * (pv.abs() + 8) * 4 * U if act != "none" else torch.zeros_like(du)
    close(db, du.sum(0), du_err.sum(0) + (SUM + (M / 256 / 4 + 16) * U) * du.abs().sum(0))
    du_r = du_err + (half(dtype) * du.abs() if act != "none" else 0.0)        # du as the products read it
    close(dx, du @ w.double(), du_r @ w.double().abs() + (N + 8) * U * (du.abs() @ w.double().abs()))
    close(dw, du.t() @ xv, du_r.t() @ xv.abs() + (M + 300) * U * (du.abs().t() @ xv.abs()))
    assert dx.dtype == dtype and dw.dtype == (dw_dtype or dtype) and db.dtype == F32 and (buf is None or dw is buf)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", LIN)
def test_linear_act_bwd(M, N, K, dtype):
    for act in ACTS:
        for ck in (False, True):
            lin_bwd_check(B(), M, N, K, dtype, act, ck, gen(M, N, K, ck), F32 if act == "lrelu" else None)


@pytest.mark.parametrize("M,N,K,dtype", [(4100, 4104, 2056, BF16), (2000, 1024, 520, BF16), (300, 264, 4096, BF16), (1000, 520, 264, F32), (33000, 264, 8, BF16)])
def test_linear_act_large_tiles(M, N, K, dtype):
    b = B()
    g = gen(M, N, K)
    x, w = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype, scale=K ** -0.5)
    bias, res = rnd(g, N, scale=0.3), rnd(g, M, N, dtype=dtype)
    y, pre = b.linear_act(x, w, bias, act="gelu_tanh", residual=res, save_pre=True)
    u = x.double() @ w.double().t() + bias.double()
    u_err = lin_bound(x, w, bias)
    v = act64(u, "gelu_tanh")[0]
    err = SLOPE * u_err + (u.abs() + 8) * 4 * U * v.abs()
    v = v + res.double()
    close(pre, u, u_err)
    close(y, v, err + U * v.abs())
    lin_bwd_check(b, M, N, K, dtype, "silu", True, gen(M, N, K, 2), F32)
    lin_bwd_check(b, M, N, K, dtype, "none", False, gen(M, N, K, 3))


# every tile, alone and split, with rows, columns and reductions that end inside one: 128 wide; 256 wide in y and dw, dx split; 256 wide over one
# step; dw split over 256 wide tiles; 128 wide and split in fp32
@pytest.mark.parametrize("M,N,K,dtype", [(2040, 2056, 2056, BF16), (1030, 8200, 2056, BF16), (5000, 2056, 8, BF16), (60000, 1016, 1024, BF16), (2056, 2056, 2056, F32)])
def test_linear_act_every_tile(M, N, K, dtype):
    b = B()
    g = gen(M, N, K, 4)
    x, w = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype, scale=K ** -0.5)
    bias, res = rnd(g, N, scale=0.3), rnd(g, M, N, dtype=dtype)
    u = x.double() @ w.double().t() + bias.double()
    u_err = lin_bound(x, w, bias)
    v = act64(u, "silu")[0]
    err = SLOPE * u_err + (u.abs() + 8) * 4 * U * v.abs()
    v = v + res.double()
    close(b.linear_act(x, w, bias, act="silu", residual=res), v, err + U * v.abs())
    r = res.clone()
    assert b.linear_act(x, w, bias, act="silu", residual=r, out=r) is r          # in place
    close(r, v, err + U * v.abs())
    del u, u_err, v, err, r
    lin_bwd_check(b, M, N, K, dtype, "gelu_tanh", False, gen(M, N, K, 5), None)
    lin_bwd_check(b, M, N, K, dtype, "none", False, gen(M, N, K, 6), F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K,ld", [(2049, 2051, 2047, 2050), (777, 201, 523, 523), (19, 70, 33, (1 << 21) + 8)])
def test_linear_odd_rows(M, N, K, ld, dtype):
    """Operands that start one element off and end inside a chunk, with faults around them; rows more than 4 MB apart."""
    b = B()
    g = gen(M, N, K, 8)

    def within(t, lead):
        buf = torch.empty(t.shape[0] * lead + 64, dtype=dtype, device=DEV)
        if buf.numel() < 1 << 24:
            buf.fill_(float("nan"))
        v = buf[1:].as_strided(t.shape, (lead, 1))
        v.copy_(t)
        return v
    x, w, dy, pre = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype, scale=K ** -0.5), rnd(g, M, N, dtype=dtype), rnd(g, M, N, dtype=dtype, scale=2.0)
    bias = rnd(g, N, scale=0.3)
    xo, wo, do = within(x, ld), within(w, K + 3), within(dy, N + 5)
    u = x.double() @ w.double().t() + bias.double()
    v = act64(u, "silu")[0]
    close(b.linear_act(xo, wo, bias, act="silu"), v, SLOPE * lin_bound(x, w, bias) + (u.abs() + 8) * 4 * U * v.abs())
    for act in ("none", "silu"):
        dx, dw, db = b.linear_act_bwd(do, xo, wo, act=act, pre=None if act == "none" else within(pre, N + 1))
        slope = act64(pre.double(), act)[1]
        du = dy.double() * slope
        du_err = dy.double().abs() * (pre.double().abs() + 8) * 4 * U if act != "none" else torch.zeros_like(du)
        close(db, du.sum(0), du_err.sum(0) + (SUM + (M / 256 / 4 + 16) * U) * du.abs().sum(0))
        du_r = du_err + (half(dtype) * du.abs() if act != "none" else 0.0)
        close(dx, du @ w.double(), du_r @ w.double().abs() + (N + 8) * U * (du.abs() @ w.double().abs()))
        close(dw, du.t() @ x.double(), du_r.t() @ x.double().abs() + (M + 300) * U * (du.abs().t() @ x.double().abs()))


def test_linear_act_bwd_long_reduction():
    lin_bwd_check(B(), 9001, 72, 136, BF16, "silu", True, gen(5), F32)
    lin_bwd_check(B(), 20000, 64, 64, F32, "none", False, gen(6))


@pytest.mark.parametrize("M", [1, 3, 4, 63, 64, 65, 129])
def test_linear_bias_gradient_of_few_rows(M):
    """One run of rows, whose sums are the gradient, and two of them; without dx and dw too."""
    b = B()
    g = gen(M, 12)
    for dtype, n in ((BF16, 200), (F32, 201)):
        dy, x, w, pre = rnd(g, M, n, dtype=dtype), rnd(g, M, 40, dtype=dtype), rnd(g, n, 40, dtype=dtype), rnd(g, M, n, dtype=dtype)
        for act in ("none", "silu"):
            du = dy.double() * act64(pre.double(), act)[1]
            err = (SUM * du.abs() + dy.double().abs() * (pre.double().abs() + 8) * 4 * U).sum(0)
            p = None if act == "none" else pre
            close(b.linear_act_bwd(dy, x, w, act=act, pre=p)[2], du.sum(0), err)
            close(b.linear_act_bwd(dy, x, w, act=act, pre=p, need=("b",))[2], du.sum(0), err)


def test_linear_gradients_against_differences():
    b = B()
    g = gen(43)
    M, N, K = 6, 10, 14
    x, w, bias, dy, res = rnd(g, M, K), rnd(g, N, K, scale=0.3), rnd(g, N), rnd(g, M, N), rnd(g, M, N)
    for act in ("none", "silu", "gelu_tanh"):
        y, pre = b.linear_act(x, w, bias, act=act, residual=res, save_pre=True)
        grads = b.linear_act_bwd(dy, x, w, act=act, pre=pre)
        f = lambda t: ((act64(t[0] @ t[1].t() + t[2], act)[0] + res.double()) * dy.double()).sum()
        args = [x.double(), w.double(), bias.double()]
        for k in range(3):
            v = torch.randn(args[k].shape, generator=g, device=DEV, dtype=F64)
            up, dn = list(args), list(args)
            h = 1e-5
            up[k], dn[k] = args[k] + h * v, args[k] - h * v
            diff = (f(up) - f(dn)) / (2 * h)
            assert abs((grads[k].double() * v).sum() - diff) <= 1e-7 * (grads[k].double() * v).abs().sum() + 40 * U * (dy.double().abs().sum() * v.abs().max() * 10)


def test_linear_layouts():
    b = B()
    g = gen(11)
    M, N, K = 70, 96, 72
    xw, ww, rw = rnd(g, M, K + 24, dtype=BF16), rnd(g, N, K + 8, dtype=BF16, scale=0.1), rnd(g, M, N + 16, dtype=BF16)
    bias = rnd(g, N)
    for off in (0, 1, 8):
        x, w, r = xw[:, off:off + K], ww[:, off % 8:off % 8 + K], rw[:, off:off + N]
        want, wpre = b.linear_act(x.contiguous(), w.contiguous(), bias, act="silu", residual=r.contiguous(), save_pre=True)
        out = torch.full((M, N + 16), 5.0, dtype=BF16, device=DEV)
        got, pre = b.linear_act(x, w, bias, act="silu", residual=r, save_pre=True, out=out[:, off:off + N])
        assert torch.equal(got, want) and torch.equal(pre, wpre)
        assert (out[:, :off] == 5).all() and (out[:, off + N:] == 5).all()
        dyw = rnd(g, M, N + 16, dtype=BF16)
        dy = dyw[:, off:off + N]
        a = b.linear_act_bwd(dy, x, w, act="silu", pre=r)
        c = b.linear_act_bwd(dy.contiguous(), x.contiguous(), w.contiguous(), act="silu", pre=r.contiguous())
        for s, t in zip(a, c):
            assert (s.float() - t.float()).abs().max() <= 2 ** -7 * t.float().abs().max()
        dww = torch.full((N, K + 16), 5.0, device=DEV)
        dw = b.linear_act_bwd(dy, x, w, act="silu", pre=r, need=("w",), dw=dww[:, off:off + K])[1]
        assert (dw.to(BF16).float() - c[1].float()).abs().max() <= 2 ** -7 * c[1].float().abs().max()
        assert (dww[:, :off] == 5).all() and (dww[:, off + K:] == 5).all()
    # the result over the residual, leading dimensions, a single row
    x, w, r = xw[:, :K].contiguous(), ww[:, :K].contiguous(), rw[:, :N].contiguous()
    want = b.linear_act(x, w, bias, act="gelu_tanh", residual=r)
    ri = r.clone()
    assert torch.equal(b.linear_act(x, w, bias, act="gelu_tanh", residual=ri, out=ri), want)
    assert torch.equal(b.linear_act(x.view(7, 10, K), w, bias, act="gelu_tanh", residual=r.view(7, 10, N)), want.view(7, 10, N))
    one = b.linear_act(x[3], w, bias, act="gelu_tanh", residual=r[3])
    assert one.shape == (N,) and (one.float() - want[3].float()).abs().max() <= 2 ** -7 * want[3].float().abs().max()
    # parts of the gradients
    dy = rnd(g, M, N, dtype=BF16)
    full = b.linear_act_bwd(dy, x, w)
    assert torch.equal(b.linear_act_bwd(dy, x, w, need=("x",))[0], full[0]) and b.linear_act_bwd(dy, x, w, need=("x",))[1:] == (None, None)
    assert torch.equal(b.linear_act_bwd(dy, x, w, need=("b",))[2], full[2])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_empty(dtype):
    b = B()
    e = lambda *s: torch.empty(*s, dtype=dtype, device=DEV)
    g = gen(9)
    z = lambda *s: rnd(g, *s, dtype=dtype)
    bias = rnd(g, 6)
    assert b.linear_act(e(0, 4), z(6, 4), bias).shape == (0, 6)
    assert b.linear_act(z(3, 4), e(0, 4)).shape == (3, 0)
    # the slope 0.01 as fp32 is off by half a step, and its product with the bias is rounded: 2 u, then the stored type's rounding
    want = act64(bias.double(), "lrelu")[0].expand(3, 6)
    close(b.linear_act(e(3, 0), e(6, 0), bias, act="lrelu"), want, 2 * U * want.abs())
    dx, dw, db = b.linear_act_bwd(e(0, 6), e(0, 4), z(6, 4), act="silu", pre=e(0, 6))
    assert dx.shape == (0, 4) and (dw == 0).all() and (db == 0).all()
    dx, dw, db = b.linear_act_bwd(e(3, 0), z(3, 4), e(0, 4))
    assert (dx == 0).all() and dx.shape == (3, 4) and dw.shape == (0, 4) and db.shape == (0,)
    dx, dw, db = b.linear_act_bwd(z(3, 6), e(3, 0), e(6, 0))
    assert dx.shape == (3, 0) and dw.shape == (6, 0) and db.shape == (6,)


def test_linear_special_values_stay_in_their_rows():
    b = B()
    g = gen(12)
    x, w = rnd(g, 40, 64, dtype=BF16), rnd(g, 48, 64, dtype=BF16)
    want = b.linear_act(x, w)
    x[5, 9], x[7, 0] = float("nan"), float("inf")
    y = b.linear_act(x, w)
    keep = torch.ones(40, dtype=torch.bool, device=DEV)
    keep[5] = keep[7] = False
    assert torch.equal(y[keep], want[keep]) and torch.isnan(y[5]).all() and not torch.isfinite(y[7]).any()
    # large pre-activations: the gates saturate without a NaN
    for act in ("silu", "gelu_tanh"):
        t = torch.tensor([[3e38, -3e38, 1e20, -1e20, 200.0, -200.0, 0.0, -0.0]], device=DEV)
        eye = torch.eye(8, device=DEV)
        v = b.linear_act(t, eye, act=act)
        assert torch.equal(v[0, :5], torch.tensor([3e38, 0, 1e20, 0, 200.0], device=DEV)) and (v[0, 5:].abs() < 1e-30).all()
        dx = b.linear_act_bwd(torch.ones(1, 8, device=DEV), t, eye, act=act, pre=t)[0]
        assert torch.equal(dx[0, [0, 2, 4]], torch.ones(3, device=DEV)) and (dx[0, [1, 3, 5]].abs() < 1e-30).all() and (dx[0, 6:] == 0.5).all()


# ---- together ------------------------------------------------------------------------------------------------------------
def block_step(b, x, p, dout):
    """A pre-norm residual block with everything kept in 8 bits, forward and backward."""
    y, mean, rstd, x8 = b.group_norm_act(x, 8, p["gamma"], p["beta"], act="silu", ckpt=True)
    h, pre = b.linear_act(y, p["w1"], p["b1"], act="gelu_tanh", save_pre=True)
    out = b.linear_act(h, p["w2"], p["b2"], residual=x)
    y8, h8, pre8 = b.ckpt8_pack(y), b.ckpt8_pack(h), b.ckpt8_pack(pre)
    dh, dw2, db2 = b.linear_act_bwd(dout, h8, p["w2"])
    dy, dw1, db1 = b.linear_act_bwd(dh, y8, p["w1"], act="gelu_tanh", pre=pre8)
    dx, dg, dbt = b.group_norm_act_bwd(dy, x8, 8, p["gamma"], p["beta"], mean, rstd, act="silu")
    return [out, dx + dout, dg, dbt, dw1, db1, dw2, db2]


def block_inputs(seed, dtype, n=6, s=16, c=64):
    g = gen(seed)
    p = dict(gamma=rnd(g, c, scale=0.2, shift=1.0), beta=rnd(g, c, scale=0.2), w1=rnd(g, 2 * c, c, dtype=dtype, scale=c ** -0.5), b1=rnd(g, 2 * c, scale=0.1),
             w2=rnd(g, c, 2 * c, dtype=dtype, scale=(2 * c) ** -0.5), b2=rnd(g, c, scale=0.1))
    return rnd(g, n, s, c, dtype=dtype), p, rnd(g, n, s, c, dtype=dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_block_with_8_bit_checkpoints_against_autograd(dtype):
    """The whole block against fp64 autograd.  What the checkpoints add: a value is off by half a step, at most 2^-7 of its block's
    largest, so a gradient is off by about 2^-7 / sqrt(3) of itself per kept tensor it passes (three of them), bf16 a further 2^-8 per
    rounding; errors of single values add with mixed signs.  2 % of the gradient's norm holds both with room."""
    b = B()
    x, p, dout = block_inputs(1, dtype)
    got = block_step(b, x, p, dout)
    leaf = {k: v.double().requires_grad_(True) for k, v in dict(p, x=x).items()}
    n, s, c = x.shape
    xg = leaf["x"].view(n, s, 8, c // 8)
    xh = ((xg - xg.mean((1, 3), keepdim=True)) / (xg.var((1, 3), unbiased=False, keepdim=True) + 1e-5).sqrt()).view(n, s, c)
    y = act64(xh * leaf["gamma"] + leaf["beta"], "silu")[0]
    h = act64(y @ leaf["w1"].t() + leaf["b1"], "gelu_tanh")[0]
    out = h @ leaf["w2"].t() + leaf["b2"] + leaf["x"]
    out.backward(dout.double())
    want = [out.detach()] + [leaf[k].grad for k in ("x", "gamma", "beta", "w1", "b1", "w2", "b2")]
    for a, t in zip(got, want):
        assert (a.double() - t).norm() <= 0.02 * t.norm()


def test_block_is_deterministic_and_runs_on_other_streams():
    b = B()
    x, p, dout = block_inputs(2, BF16, n=40)
    first = block_step(b, x, p, dout)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for st in (s1, s2, s1):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append(block_step(b, x, p, dout))
    torch.cuda.synchronize()
    for o in outs:
        for a, t in zip(o, first):
            assert torch.equal(a, t)


def test_two_captured_blocks_replayed_in_turn():
    b = B()
    sets = [block_inputs(k, BF16) for k in (3, 4)]
    eager = [block_step(b, *t) for t in sets]
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t in sets:
            block_step(b, *t)
    torch.cuda.current_stream().wait_stream(side)
    for t in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = block_step(b, *t)
        graphs.append((gr, out))
    for k in (0, 1, 1, 0, 1):
        gr, out = graphs[k]
        for o in out:
            o.fill_(float("nan"))
        gr.replay()
        again = block_step(b, *sets[1 - k])                  # eager work beside the replays
        torch.cuda.synchronize()
        for a, t in zip(out, eager[k]):
            assert torch.equal(a, t)
        for a, t in zip(again, eager[1 - k]):
            assert torch.equal(a, t)


def test_offsets_past_32_bits():
    """Row strides that put the last rows more than 2^32 bytes behind the first: one tensor of 5 GiB, few of its rows used."""
    b = B()
    ld = (1 << 31) // 8 + 8                                  # elements; 9 rows of bf16 span 4.8 GB
    big = torch.empty(9 * ld + 64, dtype=BF16, device=DEV)
    x = big.as_strided((10, 64), (ld, 1))
    g = gen(21)
    val = rnd(g, 10, 64, dtype=BF16)
    x.copy_(val)
    w, bias = rnd(g, 72, 64, dtype=BF16, scale=0.1), rnd(g, 72)
    assert torch.equal(b.linear_act(x, w, bias, act="silu"), b.linear_act(val, w, bias, act="silu"))
    dy = rnd(g, 10, 72, dtype=BF16)
    for a, t in zip(b.linear_act_bwd(dy, x, w), b.linear_act_bwd(dy, val, w)):
        assert torch.equal(a, t)
    ck, ref = b.ckpt8_pack(x), b.ckpt8_pack(val)
    assert torch.equal(ck.q, ref.q) and torch.equal(ck.e, ref.e)
    gamma, beta = rnd(g, 64), rnd(g, 64)
    a, t = b.group_norm_act(x.view(10, 1, 64), 8, gamma, beta), b.group_norm_act(val.view(10, 1, 64), 8, gamma, beta)
    for s, v in zip(a, t):
        assert torch.equal(s, v)
    d = rnd(g, 10, 1, 64, dtype=BF16)
    for s, v in zip(b.group_norm_act_bwd(d, x.view(10, 1, 64), 8, gamma, beta, t[1], t[2]), b.group_norm_act_bwd(d, val.view(10, 1, 64), 8, gamma, beta, t[1], t[2])):
        assert torch.equal(s, v)
    y = torch.empty(9 * ld + 64, dtype=BF16, device=DEV).as_strided((10, 64), (ld, 1))
    assert torch.equal(b.ckpt8_unpack(ck, out=y), b.ckpt8_unpack(ck))


def test_refusals_on_the_gpu():
    b = B()
    x, w = torch.randn(4, 8, device=DEV), torch.randn(6, 8, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        b.linear_act(x, torch.randn(8, 8, device=DEV), out=x)
    big = torch.randn(5, 6, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        b.linear_act(x, w, residual=big[:4], out=big[1:])
    with pytest.raises(ValueError, match="overlaps"):
        b.group_norm_act(x, 2, torch.ones(8, device=DEV), torch.zeros(8, device=DEV), ckpt=True, out=x)
    ones, zeros, maps = torch.ones(8, device=DEV), torch.zeros(8, device=DEV), torch.randn(3, 5, 8, device=DEV)
    with pytest.raises(ValueError, match="itself"):                               # one sample's memory for all of them
        b.group_norm_act(maps, 2, ones, zeros, out=torch.zeros(1, 5, 8, device=DEV).expand(3, 5, 8))
    with pytest.raises(ValueError, match="itself"):
        b.group_norm_act(maps, 2, ones, zeros, out=torch.zeros(64, device=DEV).as_strided((3, 5, 8), (8, 8, 1)))
    between = torch.zeros(5, 3, 8, device=DEV).transpose(0, 1)                    # samples between each other's positions: taken
    y = b.group_norm_act(maps, 2, ones, zeros, out=between)[0]
    assert y is between and torch.equal(y, b.group_norm_act(maps, 2, ones, zeros)[0])
    with pytest.raises(ValueError, match="device"):
        b.linear_act(x, w, bias=torch.randn(6))
    with pytest.raises(ValueError, match="contiguous"):
        b.linear_act(x, torch.randn(8, 6, device=DEV).t())
    with pytest.raises(ValueError, match="rows overlap"):
        b.linear_act(torch.randn(8, device=DEV).expand(4, 8), w)
    from favae_hip import lib as L
    y, out = torch.zeros(512, 2048, device=DEV), torch.zeros(128, 64, device=DEV)
    fwd = b._raw.favae_linear_act_fwd
    rc = fwd(y.data_ptr(), 2047, y.data_ptr(), 2048, None, None, 0, None, 0, out.data_ptr(), 64, 128, 64, 2048, 0, None, 0, 0, None)
    assert rc < 0 and "row stride" in L.last_error()
    assert b._raw.favae_linear_act_fwd_scratch(128, 64, 2048, 0, 0) > 0
    rc = fwd(y.data_ptr(), 2048, y.data_ptr(), 2048, None, None, 0, None, 0, out.data_ptr(), 64, 128, 64, 2048, 0, None, 0, 0, None)
    assert rc < 0 and "scratch" in L.last_error()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(17, 300, 8), (33, 201, 523), (200, 64, 64), (300, 1000, 301), (5, 7, 4096), (2000, 40, 72)])
def test_scratch_is_what_the_size_functions_say(M, N, K, dtype):
    """The C entry points with a workspace of exactly the stated size: what lies behind it stays as it was."""
    from favae_hip import lib as L
    raw = B()._raw
    g = gen(M, N, K, 77)
    code = L.F32 if dtype == F32 else L.BF16
    x, w, dy, pre = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype), rnd(g, M, N, dtype=dtype), rnd(g, M, N, dtype=dtype)
    y, dx, dw, db = torch.empty_like(dy), torch.empty_like(x), torch.empty_like(w), torch.empty(N, device=DEV)
    ck = B().ckpt8_pack(x)
    odd = int(K * x.element_size() % 16 != 0)
    odd_b = int(odd or N * x.element_size() % 16 != 0)
    st = torch.cuda.current_stream().cuda_stream

    def run(n, f):
        buf = torch.full((n + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
        L.check(f(buf.data_ptr() if n else None, n))
        assert (buf[n:] == 0xA5).all()

    run(raw.favae_linear_act_fwd_scratch(M, N, K, odd, code),
        lambda p, n: raw.favae_linear_act_fwd(x.data_ptr(), K, w.data_ptr(), K, None, None, 0, None, 0, y.data_ptr(), N, M, N, K, 2, p, n, code, st))
    for act in (0, 2):
        for xe in (None, ck):
            xp = x if xe is None else ck.q
            run(raw.favae_linear_act_bwd_scratch(M, N, K, act, int(xe is not None), odd_b, code),
                lambda p, n: raw.favae_linear_act_bwd(dy.data_ptr(), N, xp.data_ptr(), K, None if xe is None else ck.e.data_ptr(), (K + 31) // 32, w.data_ptr(),
                                                      K, pre.data_ptr(), N, None, 0, M, N, K, act, dx.data_ptr(), K, dw.data_ptr(), K, code, db.data_ptr(), p, n,
                                                      code, st))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,S,C,G", GN)
def test_group_norm_scratch_is_what_the_size_function_says(N, S, C, G, dtype):
    from favae_hip import lib as L
    raw = B()._raw
    g = gen(N, S, C, G, 78)
    code = L.F32 if dtype == F32 else L.BF16
    x, dy, gamma, beta = rnd(g, N, S, C, dtype=dtype), rnd(g, N, S, C, dtype=dtype), rnd(g, C), rnd(g, C)
    y, stat, grads = torch.empty_like(x), torch.empty(2, N, G, device=DEV), torch.empty(2, C, device=DEV)
    st = torch.cuda.current_stream().cuda_stream
    for back in (0, 1):
        n = raw.favae_gn_act_scratch(N, S, C, G, back, code)
        buf = torch.full((n + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
        p = buf.data_ptr() if n else None
        if back:
            rc = raw.favae_gn_act_bwd(dy.data_ptr(), S * C, C, x.data_ptr(), S * C, C, None, None, N, S, C, G, gamma.data_ptr(), beta.data_ptr(), stat[0].data_ptr(),
                                      stat[1].data_ptr(), 2, y.data_ptr(), S * C, C, grads[0].data_ptr(), grads[1].data_ptr(), p, n, code, st)
        else:
            rc = raw.favae_gn_act_fwd(x.data_ptr(), S * C, C, N, S, C, G, gamma.data_ptr(), beta.data_ptr(), 1e-5, 2, y.data_ptr(), S * C, C, stat[0].data_ptr(),
                                      stat[1].data_ptr(), None, None, p, n, code, st)
        L.check(rc)
        assert (buf[n:] == 0xA5).all()


# ---- checkpoints of the forward pass, further shapes ------------------------------------------------------------------------
# groups wider than a workgroup: whole vectors but no whole blocks of 32 channels wide (4104, 2056, 4112), off the vector grid, whole blocks (8192)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,S,C,G", [(2, 16, 16416, 4), (2, 16, 16416, 8), (2, 5, 8224, 4), (2, 5, 8224, 2), (1, 3, 8224, 1), (1, 3, 12299, 1), (2, 5, 8192, 1)])
def test_group_norm_checkpoint_of_wide_groups_is_the_input_packed(N, S, C, G, dtype):
    b = B()
    # every channel of another size, so that neighbouring blocks have other steps
    x = (rnd(gen(31, N, C, G), N, S, C) * torch.exp2(torch.randint(-12, 12, (C,), generator=gen(32, C), device=DEV).float())).to(dtype)
    ck = b.group_norm_act(x, G, torch.ones(C, device=DEV), torch.zeros(C, device=DEV), act="silu", ckpt=True)[3]
    ref = b.ckpt8_pack(x)
    assert torch.equal(ck.e, ref.e) and torch.equal(ck.q, ref.q)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,C,G", [(2, 8192, 1), (2, 4099, 1), (3, 16416, 2), (1, 1 << 20, 4)])
def test_group_norm_of_no_positions_in_wide_groups(N, C, G, dtype):
    """Mean 0 and variance 0, also where a group is wider than a workgroup."""
    b = B()
    e, one, zero = torch.empty(N, 0, C, dtype=dtype, device=DEV), torch.ones(C, device=DEV), torch.zeros(C, device=DEV)
    for eps in (1e-5, 1.0):
        y, m, r = b.group_norm_act(e, G, one, zero, eps=eps)
        assert y.shape == e.shape and (m == 0).all()
        close(r, torch.full((N, G), eps, device=DEV, dtype=F64).rsqrt(), 3 * U * eps ** -0.5)      # eps as fp32, the root and the division
    dx, dg, db = b.group_norm_act_bwd(e, e, G, one, zero, m, r)
    assert dx.shape == e.shape and (dg == 0).all() and (db == 0).all()


def checkpoint_layouts(g, C, dtype):
    wide = rnd(g, 5, 12, C + 24, dtype=dtype)
    one = rnd(g, 1, 7, C, dtype=dtype)
    return {"cropped": wide[:, 2:9, :C], "cropped and shifted": wide[:, :7, 3:C + 3], "every other sample": wide[::2, :, :C], "one position": wide[:, 4, :C],
            "one sample for all": one.expand(4, 7, C), "one position for all": one[:, :1].expand(4, 1, C), "one row for all": one[0, 0].expand(4, C),
            "samples between each other's positions": wide.transpose(0, 1)[:7, :, :C]}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("C,G", [(40, 5), (64, 8), (33, 3), (4104, 1)])
def test_group_norm_checkpoint_of_any_layout(C, G, dtype):
    b = B()
    gamma, beta = torch.ones(C, device=DEV), torch.zeros(C, device=DEV)
    for name, x in checkpoint_layouts(gen(33, C), C, dtype).items():
        y, m, r, ck = b.group_norm_act(x, G, gamma, beta, act="silu", ckpt=True)
        ref = b.ckpt8_pack(x.contiguous())
        assert torch.equal(ck.q, ref.q) and torch.equal(ck.e, ref.e), name
        want, m2, r2, z, z_err, m_err, r_rel = gn_ref(x.contiguous(), gamma, beta, G, "silu")
        close(y.reshape(want.shape), want, SLOPE * z_err + (z.abs() + 8) * 4 * U * want.abs())
        close(m, m2, m_err)


@pytest.mark.parametrize("C,G", [(64, 8), (72, 9), (66, 3)])
def test_group_norm_checkpoint_makes_no_copy_of_its_input(C, G):
    """A cropped map with a checkpoint: outputs, checkpoint and workspace are all that is allocated."""
    b = B()
    wide = rnd(gen(34), 64, 33, 32, C + 24, dtype=BF16)
    x = wide[:, :32, :, :C].flatten(1, 2)
    assert x.data_ptr() == wide.data_ptr() and not x.is_contiguous() and x.stride(0) != 1024 * x.stride(1)
    gamma, beta = torch.ones(C, device=DEV), torch.zeros(C, device=DEV)
    b.group_norm_act(x, G, gamma, beta, act="silu", ckpt=True)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = b.group_norm_act(x, G, gamma, beta, act="silu", ckpt=True)
    held = torch.cuda.memory_allocated() - before
    assert torch.cuda.max_memory_allocated() - before - held < x.numel()       # half of what a copy takes
    del out


def test_sizes_past_a_limit_are_value_errors():
    """What only the library refuses arrives as the errors of wrong arguments do, and as the library's own."""
    from favae_hip import lib as L
    b = B()
    k = (1 << 20) + 8
    x, w = torch.zeros(2, k, dtype=BF16, device=DEV), torch.zeros(3, k, dtype=BF16, device=DEV)
    c = (1 << 24) + 8
    m, v = torch.zeros(1, 1, c, dtype=BF16, device=DEV), torch.zeros(c, device=DEV)
    st = torch.zeros(1, 1, device=DEV)
    for call, text in ((lambda: b.linear_act(x, w), "too large"), (lambda: b.linear_act_bwd(torch.zeros(2, 3, dtype=BF16, device=DEV), x, w), "too large"),
                       (lambda: b.group_norm_act(m, 1, v, v), "too large"), (lambda: b.group_norm_act_bwd(m, m, 1, v, v, st, st), "too large")):
        for err in (ValueError, L.FavaeHipError):
            with pytest.raises(err, match=text):
                call()


def test_a_lost_gradient_is_an_error():
    """Inputs that require gradients: the values are those of no_grad, and differentiating them says where the gradients are instead of leaving them out."""
    b = B()
    g = gen(51)
    x, w = rnd(g, 6, 5, 32), torch.nn.Parameter(rnd(g, 24, 32))
    gamma, beta, bias, res = torch.nn.Parameter(rnd(g, 32)), rnd(g, 32), rnd(g, 24), rnd(g, 6, 5, 24)
    norm = lambda **k: b.group_norm_act(x, 4, gamma, beta, act="silu", **k)
    lin = lambda **k: b.linear_act(x, w, bias, act="silu", **k)
    with torch.no_grad():
        want = list(norm()) + list(lin(save_pre=True)) + [lin()]
    assert not any(t.requires_grad for t in want)
    got = list(norm(ckpt=True)[:3]) + list(lin(save_pre=True)) + [lin()]
    for k, (a, t) in enumerate(zip(got, want)):
        assert torch.equal(a, t) and a.dtype == t.dtype
        with pytest.raises(RuntimeError, match="group_norm_act_bwd" if k < 3 else "linear_act_bwd"):
            (2 * a).sum().backward()
    assert w.grad is None and gamma.grad is None
    for t in (x, beta):
        t.requires_grad_(True)
    with pytest.raises(RuntimeError, match="linear_act_bwd"):
        b.linear_act(x, w.detach()).sum().backward()
    with pytest.raises(RuntimeError, match="linear_act_bwd"):
        b.linear_act(x.detach(), w.detach(), residual=res.clone().requires_grad_(True)).sum().backward()
    with pytest.raises(RuntimeError, match="group_norm_act_bwd"):
        b.group_norm_act(x.detach(), 4, gamma.detach(), beta)[0].sum().backward()
    # an output of the caller's, as with torch's own operators
    buf, y = torch.empty(6, 5, 24, device=DEV), torch.empty(6, 5, 32, device=DEV)
    for call in (lambda: lin(out=buf), lambda: norm(out=y)):
        with pytest.raises(ValueError, match="out"):
            call()
    with torch.no_grad():
        assert lin(out=buf) is buf and torch.equal(buf, want[5]) and norm(out=y)[0] is y and torch.equal(y, want[0])
    # gradients are constants, and so is what was packed
    grads = b.linear_act_bwd(res, x, w)
    assert not any(t.requires_grad for t in grads) and not b.ckpt8_unpack(b.ckpt8_pack(x)).requires_grad


def test_operators_inside_an_autograd_function():
    b = B()
    g = gen(52)

    class Linear(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, bias):
            y, pre = b.linear_act(x, w, bias, act="silu", save_pre=True)
            ctx.save_for_backward(x, w, pre)
            return y

        @staticmethod
        def backward(ctx, dy):
            x, w, pre = ctx.saved_tensors
            return b.linear_act_bwd(dy, x, w, act="silu", pre=pre)
    x, w, bias = rnd(g, 20, 32).requires_grad_(True), rnd(g, 24, 32).requires_grad_(True), rnd(g, 24).requires_grad_(True)
    dy = rnd(g, 20, 24)
    Linear.apply(x, w, bias).backward(dy)
    pre = b.linear_act(x.detach(), w.detach(), bias.detach(), act="silu", save_pre=True)[1]
    for a, t in zip((x, w, bias), b.linear_act_bwd(dy, x.detach(), w.detach(), act="silu", pre=pre)):
        assert torch.equal(a.grad, t)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_outputs_into_other_columns_of_the_input_s_buffer(dtype):
    b = B()
    g = gen(61)
    start = rnd(g, 4, 9, 80, dtype=dtype)
    gamma, beta, w = rnd(g, 32), rnd(g, 32), rnd(g, 40, 32, dtype=dtype, scale=0.2)
    for off in (32, 37):
        big = start.clone()
        y = b.group_norm_act(big[..., :32], 4, gamma, beta, act="silu", out=big[..., off:off + 32])[0]
        assert torch.equal(y, b.group_norm_act(start[..., :32].clone(), 4, gamma, beta, act="silu", out=torch.empty_like(start)[..., off:off + 32])[0])
        z = b.linear_act(big[..., :32], w, act="silu", out=big[..., off:off + 40])
        assert torch.equal(z, b.linear_act(start[..., :32], w, act="silu"))
        ck = b.ckpt8_pack(start[..., :32])
        b.ckpt8_unpack(ck, out=big[..., off:off + 32])
        assert torch.equal(big[..., :32], start[..., :32]) and torch.equal(big[..., off + 40:], start[..., off + 40:])


# ---- every form of the norm --------------------------------------------------------------------------------------------------
# Each kernel variant that the rules choose between (test_cpu_blocks.py holds the list to it), in both types: wave with 1, 2, 4, 8 vectors a lane and 1 to
# 8 groups a vector; held with up to 4, 8, 12, 16 vectors a thread; piped with 1 to 8 groups a vector; chunked; last channel blocks that are partial,
# positions that are no multiple of what a workgroup takes at once, samples that workgroups take unequal numbers of.
GN_FORMS = [(1, 1, 24, 12), (1, 1, 24, 6), (1, 5, 40, 5), (1, 9, 40, 20), (1, 5, 72, 9), (1, 11, 432, 9), (1, 1, 12, 12), (1, 131, 24, 12), (1, 140, 24, 3),
            (1, 17, 16, 16), (1, 33, 16, 16), (1, 348, 33, 11), (1, 151, 16, 16), (1, 518, 8, 8), (1, 5, 40, 20), (1, 5, 80, 20), (1, 9, 72, 9), (1, 17, 40, 20),
            (1, 9, 80, 20), (1, 344, 72, 3), (1, 144, 24, 6), (1, 44, 60, 20), (1, 1031, 40, 20), (1, 33, 32, 32), (1, 2140, 1, 1), (1, 237, 35, 5),
            (72, 2061, 1, 1), (1, 9, 20, 20), (1, 17, 20, 20), (1, 131, 12, 12), (1, 132, 12, 6), (1, 142, 12, 3), (1, 25, 240, 20), (72, 1313, 1, 1),
            (34, 1049, 44, 11), (1, 698, 35, 5), (33, 85, 216, 9), (25, 1055, 64, 64), (1, 513, 96, 3), (20, 1698, 72, 9), (1, 1067, 80, 20), (32, 1257, 15, 3),
            (12, 205, 320, 64), (306, 281, 40, 20), (297, 284, 40, 5), (32, 426, 35, 5), (98, 1549, 16, 16), (558, 291, 16, 16), (21, 1119, 72, 9), (37, 693, 35, 5),
            (236, 261, 80, 20), (68, 102, 100, 20), (20, 1780, 36, 9), (275, 279, 20, 20), (126, 85, 240, 20), (266, 211, 60, 20), (177, 303, 100, 20),
            (4999, 2, 32, 8)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,S,C,G", GN_FORMS)
def test_group_norm_every_form(N, S, C, G, dtype):
    b = B()
    g = gen(N, S, C, G, 5)
    x = rnd(g, N, S, C, dtype=dtype, scale=1.7, shift=3.0)
    gamma, beta = rnd(g, C, scale=0.3, shift=1.0), rnd(g, C, scale=0.5)
    for act in ACTS:
        want, m, r, z, z_err, m_err, r_rel = gn_ref(x, gamma, beta, G, act)
        for ckpt in (False, True):
            y, mean, rstd, *ck = b.group_norm_act(x, G, gamma, beta, act=act, ckpt=ckpt)
            close(mean, m, m_err)
            close(rstd, r, r * r_rel)
            close(y, want, SLOPE * z_err + (z.abs() + 8) * 4 * U * want.abs())
            if ckpt:
                ref = b.ckpt8_pack(x)
                assert torch.equal(ck[0].q, ref.q) and torch.equal(ck[0].e, ref.e)
    for act in ACTS:
        for ck in (False, True):
            gn_bwd_check(b, N, S, C, G, dtype, act, ck, gen(N, S, C, G, 6 + ck))


# the piped backward: 1, 2, 4 and 8 groups a vector, 8 vectors a thread, unequal numbers of samples
@pytest.mark.parametrize("dtype,N,S,C,G", [(F32, 275, 279, 20, 20), (F32, 306, 281, 40, 20), (F32, 297, 284, 40, 5), (F32, 600, 101, 128, 1), (F32, 300, 500, 64, 8),
                                           (BF16, 558, 291, 16, 16), (BF16, 306, 281, 40, 20), (BF16, 236, 261, 80, 20), (BF16, 297, 284, 40, 5),
                                           (BF16, 600, 101, 256, 1), (BF16, 300, 1000, 64, 8)])
def test_group_norm_piped_backward(dtype, N, S, C, G):
    b = B()
    g = gen(N, S, C, G, 8)
    pad = 16 // torch.finfo(dtype).bits * 8                    # elements of 16 bytes
    wide = rnd(g, N, S + 1, C + pad, dtype=dtype, scale=1.7, shift=3.0)
    x, dy = wide[:, :S, :C], rnd(g, N, S + 2, C + 2 * pad, dtype=dtype)[:, 1:S + 1, pad:C + pad]
    gamma, beta = rnd(g, C, scale=0.3, shift=1.0), rnd(g, C, scale=0.5)
    mean, rstd = b.group_norm_act(x, G, gamma, beta, act="silu")[1:]
    ck = b.ckpt8_pack(x.contiguous())
    for src in (x, ck):
        one = b.group_norm_act_bwd(dy.contiguous(), x.contiguous() if src is x else ck, G, gamma, beta, mean, rstd, act="silu")
        # strided rows, the gradient over dy, into rows with others between them: the same kernel, the same bits
        buf = torch.full((N, S + 1, C + pad), 7.0, dtype=dtype, device=DEV)
        for out in (None, dy.clone(), buf[:, :S, :C]):
            d = out if out is not None and out.is_contiguous() else dy
            two = b.group_norm_act_bwd(d, src, G, gamma, beta, mean, rstd, act="silu", out=out)
            assert out is None or two[0] is out
            for a, t in zip(two, one):
                assert torch.equal(a, t)
        assert (buf[:, S:] == 7).all() and (buf[..., C:] == 7).all()
    # a fault stays in its sample and group, and in the groups that share its block of a checkpoint
    cg = C // G
    x = x.contiguous()
    for n, i, c in ((N - 1, S - 1, C - 1), (N // 2, 0, 0), (N // 3, S // 2, (G // 2) * cg)):
        x[n, i, c] = float("nan")
    ck = b.ckpt8_pack(x)
    mean, rstd = b.group_norm_act(x, G, gamma, beta, act="silu")[1:]
    assert torch.isnan(mean).sum() == 3
    for src, v in ((x, x), (ck, b.ckpt8_unpack(ck))):
        dx, dg, db = b.group_norm_act_bwd(dy, src, G, gamma, beta, mean, rstd, act="silu")
        z = torch.isnan(v) | torch.isnan(mean).repeat_interleave(cg, 1)[:, None, :]
        bad = z.reshape(N, S, G, cg).any(3).any(1).repeat_interleave(cg, 1)[:, None, :].expand(N, S, C)
        assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()
        cols = z.any(0).any(0)
        for t in (dg, db):
            assert torch.isnan(t[cols]).all() and torch.isfinite(t[~cols]).all()


# 128-wide fp32 tiles alone (y; dx; dw), and in bf16 128-wide ones split (dw), 64-wide ones split with two stages (dx; y)
@pytest.mark.parametrize("M,N,K,dtype", [(4311, 1080, 4, F32), (2638, 4, 1657, F32), (19, 1418, 2903, F32), (5201, 73, 2073, BF16), (1484, 2568, 5, BF16),
                                         (2638, 4, 1657, BF16)])
def test_linear_act_tiles_alone_and_split(M, N, K, dtype):
    b = B()
    g = gen(M, N, K, 13)
    x, w = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype, scale=K ** -0.5)
    bias, res = rnd(g, N, scale=0.3), rnd(g, M, N, dtype=dtype)
    y, pre = b.linear_act(x, w, bias, act="gelu_tanh", residual=res, save_pre=True)
    u = x.double() @ w.double().t() + bias.double()
    u_err = lin_bound(x, w, bias)
    v = act64(u, "gelu_tanh")[0]
    err = SLOPE * u_err + (u.abs() + 8) * 4 * U * v.abs()
    v = v + res.double()
    close(pre, u, u_err)
    close(y, v, err + U * v.abs())
    for ck in (False, True):
        lin_bwd_check(b, M, N, K, dtype, "silu", ck, gen(M, N, K, 14 + ck))
    lin_bwd_check(b, M, N, K, dtype, "none", False, gen(M, N, K, 16), F32)


@pytest.mark.parametrize("M,N,K", [(65536, 1024, 1024), (16384, 4096, 1024)])
def test_large_product_gradients_repeat_bit_for_bit(M, N, K):
    """Ring of tiles, split reductions and their joins at full size, other work between the runs."""
    b = B()
    g = gen(M, N, K, 17)
    dy, x, pre, w = rnd(g, M, N, dtype=BF16), rnd(g, M, K, dtype=BF16), rnd(g, M, N, dtype=BF16), rnd(g, N, K, dtype=BF16, scale=K ** -0.5)
    x8, pre8 = b.ckpt8_pack(x), b.ckpt8_pack(pre)
    for src, p in ((x, pre), (x8, pre8)):
        first = b.linear_act_bwd(dy, src, w, act="gelu_tanh", pre=p)
        for _ in range(4):
            b.linear_act(x, w, act="silu")
            for a, t in zip(b.linear_act_bwd(dy, src, w, act="gelu_tanh", pre=p), first):
                assert torch.equal(a, t)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,S,C,G", [(200, 1500, 32, 4), (24, 512, 256, 32), (48, 2048, 64, 8)])
def test_group_norm_checkpoint_on_either_side_of_its_limit(N, S, C, G, dtype):
    b = B()
    g = gen(N, S, C, G, 18)
    x = rnd(g, N, S, C, dtype=dtype, scale=1.7, shift=3.0)
    gamma, beta = rnd(g, C, scale=0.3, shift=1.0), rnd(g, C, scale=0.5)
    y, mean, rstd, ck = b.group_norm_act(x, G, gamma, beta, act="silu", ckpt=True)
    want, m, r, z, z_err, m_err, r_rel = gn_ref(x, gamma, beta, G, "silu")
    close(mean, m, m_err)
    close(rstd, r, r * r_rel)
    close(y, want, SLOPE * z_err + (z.abs() + 8) * 4 * U * want.abs())
    ref = b.ckpt8_pack(x)
    assert torch.equal(ck.q, ref.q) and torch.equal(ck.e, ref.e)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,S,C,G", [(64, 1024, 64, 8), (200, 1500, 32, 4), (3, 64, 64, 8), (2, 16, 16416, 4), (5, 195, 210, 30), (2, 4096, 64, 16), (300, 500, 64, 8),
                                     (1, 20000, 33, 3)])
def test_group_norm_scratch_with_a_checkpoint_and_with_odd_rows(N, S, C, G, dtype):
    """As above, for the forward pass with a checkpoint and for rows that are not 16-byte aligned, whose forms differ; the checkpoint's own ends too."""
    from favae_hip import lib as L
    raw = B()._raw
    g = gen(N, S, C, G, 79)
    code = L.F32 if dtype == F32 else L.BF16
    nb = (C + 31) // 32
    st = torch.cuda.current_stream().cuda_stream
    gamma, beta = rnd(g, C), rnd(g, C)
    for lead in (0, 1):                                        # elements before the first
        x, dy, y = (rnd(g, N * S * C + 1, dtype=dtype)[lead:lead + N * S * C] for _ in range(3))
        stat, grads = torch.empty(2, N, G, device=DEV), torch.empty(2, C, device=DEV)
        q, e = torch.full((N * S * C + 64,), 9, dtype=torch.int8, device=DEV), torch.full((N * S * nb + 64,), 9, dtype=torch.uint8, device=DEV)
        for back in (0, 1):
            n = raw.favae_gn_act_scratch(N, S, C, G, back, code)
            buf = torch.full((n + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
            p = buf.data_ptr() if n else None
            if back:
                rc = raw.favae_gn_act_bwd(dy.data_ptr(), S * C, C, x.data_ptr(), S * C, C, None, None, N, S, C, G, gamma.data_ptr(), beta.data_ptr(),
                                          stat[0].data_ptr(), stat[1].data_ptr(), 2, y.data_ptr(), S * C, C, grads[0].data_ptr(), grads[1].data_ptr(), p, n, code, st)
            else:
                rc = raw.favae_gn_act_fwd(x.data_ptr(), S * C, C, N, S, C, G, gamma.data_ptr(), beta.data_ptr(), 1e-5, 2, y.data_ptr(), S * C, C,
                                          stat[0].data_ptr(), stat[1].data_ptr(), q.data_ptr(), e.data_ptr(), p, n, code, st)
            L.check(rc)
            assert (buf[n:] == 0xA5).all() and (q[N * S * C:] == 9).all() and (e[N * S * nb:] == 9).all()
        ref = B().ckpt8_pack(x.view(N * S, C))
        assert torch.equal(q[:N * S * C].view(N * S, C), ref.q) and torch.equal(e[:N * S * nb].view(N * S, nb), ref.e)


def test_the_node_that_raises_keeps_no_parameter():
    """An output that lives on holds no node of the caller's leaves: their gradients may be captured into a graph meanwhile."""
    b = B()
    g = gen(53)
    x, w = rnd(g, 6, 32).requires_grad_(True), torch.nn.Parameter(rnd(g, 24, 32))
    gamma, beta = torch.nn.Parameter(rnd(g, 32)), rnd(g, 32)
    mine = [x, w, gamma]
    for y in (b.linear_act(x, w), b.group_norm_act(x.view(1, 6, 32), 4, gamma, beta)[0]):
        todo, seen = [y.grad_fn], 0
        while todo:
            node = todo.pop()
            seen += 1
            assert not any(getattr(node, "variable", None) is t for t in mine)
            todo += [f for f, _ in node.next_functions if f is not None]
        assert seen
    # and the calls are captured in grad mode as they are under no_grad
    want = b.linear_act(x.detach(), w.detach(), act="silu")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.linear_act(x, w, act="silu")
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        y = b.linear_act(x, w, act="silu")
    for _ in range(3):
        y.detach().fill_(float("nan"))
        graph.replay()
        assert torch.equal(y, want)
