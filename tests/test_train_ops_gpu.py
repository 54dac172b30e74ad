"""GPU: training through frozen int4 weights (activations kept in 8 bits, the adapter's gradients from them, the input
gradient, softmax cross entropy over a vocabulary) against 64-bit restatements.

Tolerances.  S = sum |a||b| over a product's terms, in 64 bits.
  fp32: operands to 2^-21, and sums of rounded terms whose chains are at most 255 long: |error| <= 2^-16 S.
  bf16: one operand rounded to f16 (2^-11 of each term), the result to bf16 (2^-8 of it): 2^-11 S + 2^-8 |y| + 2^-16 S.
Logits are held to the fp32 bound for both types: dz = 2^-16 max_v S (bf16 rows are exact and W enters as f16 hi and lo).
Then lse is off by dz + 2^-20 (1 + |lse|), a loss by twice that, a probability by 2 dz + 2^-16 of itself.
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from spaceslug_b200 import synth

pytestmark = pytest.mark.gpu
DT = ("f32", "bf16")


@pytest.fixture(autouse=True)
def _seed():
    import torch
    torch.manual_seed(1234)


def _dt(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


def _w64(packed, scales, k, n, cuda):
    """W [k, n] in 64 bits from the layout's bytes."""
    import torch
    by = torch.from_numpy(np.ascontiguousarray(packed).view(np.uint8).reshape(n, k // 2)).to(cuda).to(torch.int64)
    v = torch.stack((by % 16, by // 16), -1).flatten(1)
    v = torch.where(v > 7, v - 16, v).double()
    sc = torch.from_numpy(np.ascontiguousarray(scales).reshape(n, k // 32)).to(cuda).double()
    return (v * sc.repeat_interleave(32, 1)).T


def _weights(k, n, seed, lo=0.005, hi=0.02):
    _, packed, scales = synth.make_weights(k, n, lo, hi, seed=seed)
    return packed, scales


def _randn(shape, cuda, seed):
    import torch
    return torch.randn(shape, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed))


# ---------------------------------------------------------------------------------------------------- 8-bit copies --
def _act8_oracle(x):
    """codes and step bytes of fp32 numpy [m, k] by exact 64-bit arithmetic."""
    m, k = x.shape
    g = x.astype(np.float64).reshape(m, k // 32, 32)
    top = np.abs(g).max(-1)
    e = np.full(top.shape, -126, np.int64)
    fin = np.isfinite(top)
    while True:  # the smallest e >= -126 with top <= 127 2^e
        more = fin & (top > 127.0 * np.exp2(e.astype(np.float64)))
        if not more.any():
            break
        e[more] += 1
    codes = np.where(fin[..., None], np.rint(np.where(fin[..., None], g, 0.0) / np.exp2(e.astype(np.float64))[..., None]), 0)
    codes = np.where((e == 122)[..., None], np.clip(codes, -63, 63), codes)  # 64 * 2^122 is no fp32 value
    return codes.reshape(m, k).astype(np.int8), np.where(fin, e + 127, 255).astype(np.uint8)


def _act8(session, x, dtype):
    import torch
    m, k = x.shape
    codes = torch.full((m, k), 77, dtype=torch.int8, device=x.device)
    exps = torch.full((m, k // 32), 99, dtype=torch.uint8, device=x.device)
    session.act8_pack_device(x.data_ptr(), codes.data_ptr(), exps.data_ptr(), m, k, dtype=dtype)
    back = torch.empty_like(x)
    session.act8_unpack_device(codes.data_ptr(), exps.data_ptr(), back.data_ptr(), m, k, dtype=dtype)
    return codes, exps, back


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k", [(1, 32), (3, 64), (1, 4096), (129, 4128), (7, 11008)])
def test_act8_is_the_exact_rounding(session, cuda, m, k, dtype):
    import torch
    x = (_randn((m, k), cuda, m + k) * torch.exp2(torch.randint(-20, 20, (m, k // 32), device=cuda).float())
         .repeat_interleave(32, 1)).to(_dt(dtype))
    codes, exps, back = _act8(session, x, dtype)
    c, e = _act8_oracle(x.float().cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), c) and np.array_equal(exps.cpu().numpy(), e)
    step = np.exp2(e.astype(np.float64) - 127).repeat(32, 1)
    assert np.array_equal(back.double().cpu().numpy(), c * step)  # exact in both types
    assert np.all(np.abs(back.double().cpu().numpy() - x.double().cpu().numpy()) <= step / 2)


def test_act8_edges(session, cuda):
    """Borders of the step rule, zeros, the smallest and largest magnitudes, infinities and NaN (their group alone)."""
    import torch
    rows = np.zeros((12, 64), np.float32)
    rows[0, :3] = 127.0, -127.0, 0.5
    rows[1, :3] = np.nextafter(np.float32(127.0), np.float32(200.0)), 1.0, 3.0
    rows[2, :2] = 127.0 * 2.0 ** -40, 2.0 ** -41
    rows[3, :2] = np.finfo(np.float32).max, 1.0
    rows[4, :2] = 2.0 ** -140, -(2.0 ** -126)  # below the least step's half, and one step
    rows[5, 1], rows[5, 40] = np.inf, 3.0
    rows[6, 33], rows[6, 2] = np.nan, -5.0
    rows[7, 5], rows[7, 6] = -np.inf, np.inf
    rows[8, :4] = 64.0, 63.5, 62.5, -61.5  # ties go to even codes
    rows[9, :] = -0.0
    rows[10, :32] = 1e-38
    rows[11, :] = 2.0 ** 100
    x = torch.from_numpy(rows).to(cuda)
    codes, exps, back = _act8(session, x, "f32")
    c, e = _act8_oracle(rows)
    assert np.array_equal(codes.cpu().numpy(), c) and np.array_equal(exps.cpu().numpy(), e)
    b = back.cpu().numpy()
    bad = np.repeat(e == 255, 32, 1)
    assert bad.sum() == 3 * 32 and np.isnan(b[bad]).all()
    assert np.array_equal(b[~bad].astype(np.float64), (c * np.exp2(e.astype(np.float64) - 127).repeat(32, 1))[~bad])


# ------------------------------------------------------------------------------------------- gradients of the adapter --
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k,n,rank,c0,c1", [
    (1, 64, 256, 4, 0, 256), (33, 512, 700, 5, 100, 600), (128, 256, 160, 8, 0, 160), (300, 1024, 704, 64, 0, 704),
    (257, 2080, 1001, 33, 0, 1001), (515, 4096, 640, 16, 32, 616), (128, 32, 32, 1, 0, 32),
    (1500, 1056, 2048, 32, 0, 2048), (30, 1248, 23, 1, 0, 23), (130, 3520, 1, 17, 0, 1), (77, 96, 1003, 3, 500, 513)])
def test_backward_from_8_bits(session, cuda, m, k, n, rank, c0, c1, dtype):
    import torch
    packed, scales = _weights(k, n, 3)
    rng = np.random.default_rng(m + n)
    A = (rng.standard_normal((k, rank)) * 0.02).astype(np.float32)
    B = (rng.standard_normal((rank, n)) * 0.02).astype(np.float32)
    x = _randn((m, k), cuda, 1)
    dy = _randn((m, c1 - c0), cuda, 2).to(_dt(dtype))
    codes, exps, back = _act8(session, x, "f32")
    da = torch.full((k, rank), float("nan"), device=cuda)
    db = torch.full((rank, c1 - c0), float("nan"), device=cuda)
    with session.weights(packed, scales, k, n, c0, c1) as h:
        h.set_lora(A, B, 2.0 * rank)
        args = (codes.data_ptr(), exps.data_ptr(), dy.data_ptr(), m)
        h.lora_backward_act8(*args, dtype=dtype, da=da.data_ptr(), db=db.data_ptr())
        _, _, ha, hb = h.get_lora(rank, grads=True)
        h.lora_backward_act8(*args, dtype=dtype)
        _, _, ha2, hb2 = h.get_lora(rank, grads=True)
    assert np.array_equal(ha, da.cpu().numpy()) and np.array_equal(hb, db.cpu().numpy())
    assert np.array_equal(ha, ha2) and np.array_equal(hb, hb2)  # sums in a fixed order
    X, D = back.double(), dy.double()
    A64, B64 = torch.from_numpy(A).to(cuda).double(), torch.from_numpy(np.ascontiguousarray(B[:, c0:c1])).to(cuda).double()
    for got, ref, S in ((da, 2.0 * X.T @ (D @ B64.T), 2.0 * X.abs().T @ (D.abs() @ B64.abs().T)),
                        (db, 2.0 * (X @ A64).T @ D, 2.0 * (X.abs() @ A64.abs()).T @ D.abs())):
        # two chained products, each to 2^-16 of its S
        assert ((got.double() - ref).abs() <= 2 * 2.0 ** -16 * S).all()
        assert (got.double() - ref).norm() <= 1e-5 * ref.norm()
    assert session.device_status(0) == 0


def test_backward_from_8_bits_spreads_nan_and_steps(session, cuda):
    """A NaN group of X reaches its 32 rows of dA and (through T) dB, no other row of dA; groups whose steps are far
    apart stay exact."""
    import torch
    m, k, n, rank = 160, 256, 96, 8
    packed, scales = _weights(k, n, 5)
    A, B = np.full((k, rank), 0.01, np.float32), np.full((rank, n), 0.02, np.float32)
    x = _randn((m, k), cuda, 3) * torch.exp2(torch.randint(-30, 30, (k // 32,), device=cuda).float()).repeat_interleave(32)
    clean = x.clone()
    x[7, 70] = float("nan")
    dy = _randn((m, n), cuda, 4)
    out = []
    with session.weights(packed, scales, k, n) as h:
        h.set_lora(A, B, float(rank))
        for v in (clean, x):
            codes, exps, _ = _act8(session, v, "f32")
            h.lora_backward_act8(codes.data_ptr(), exps.data_ptr(), dy.data_ptr(), m)
            out.append(h.get_lora(rank, grads=True)[2:])
        codes, exps, back = _act8(session, clean, "f32")
    # two chained products, each to 2^-16 of its S (a row's terms may cancel: S, not the result, bounds the error)
    B64 = torch.from_numpy(B).to(cuda).double()
    ref = (back.double().T @ (dy.double() @ B64.T)).cpu().numpy()
    S = (back.double().abs().T @ (dy.double().abs() @ B64.abs().T)).cpu().numpy()
    assert np.all(np.abs(out[0][0] - ref) <= 2 * 2.0 ** -16 * S)
    assert np.isnan(out[1][0][64:96]).all() and np.isnan(out[1][1]).all()
    keep = np.r_[0:64, 96:256]
    assert np.array_equal(out[1][0][keep], out[0][0][keep])


@pytest.mark.parametrize("m,n", [(30, 23), (130, 1001), (5, 1), (64, 130)])
def test_fp32_backward_with_rows_of_any_length(session, cuda, m, n):
    """The fp32 backward where dY's rows are no whole 16 bytes: nothing behind a row (here NaN behind the last) takes
    part.  dY and its last row's neighbour are one buffer, so nothing is read out of range either way."""
    import torch
    k, rank = 160, 4
    packed, scales = _weights(k, n, 37)
    rng = np.random.default_rng(n)
    A, B = (rng.standard_normal(s).astype(np.float32) * 0.02 for s in ((k, rank), (rank, n)))
    x = _randn((m, k), cuda, 1)
    buf = torch.full((m * n + 4,), float("nan"), device=cuda)
    dy = buf[:m * n].view(m, n)
    dy.copy_(_randn((m, n), cuda, 2))
    with session.weights(packed, scales, k, n) as h:
        h.set_lora(A, B, float(rank))
        h.lora_backward(x.data_ptr(), dy.data_ptr(), m)
        _, _, da, db = h.get_lora(rank, grads=True)
    X, D, A64, B64 = x.double(), dy.double(), torch.from_numpy(A).to(cuda).double(), torch.from_numpy(B).to(cuda).double()
    for got, ref, S in ((da, X.T @ (D @ B64.T), X.abs().T @ (D.abs() @ B64.abs().T)),
                        (db, (X @ A64).T @ D, (X.abs() @ A64.abs()).T @ D.abs())):
        assert ((torch.from_numpy(got).to(cuda).double() - ref).abs() <= 2 * 2.0 ** -16 * S).all()


# ------------------------------------------------------------------------------------------------------ dX of a layer --
def _check_dx(got, dtype, ref, S):
    import torch
    err = (got.double() - ref).abs()
    tol = 2.0 ** -16 * S + 1e-37
    if dtype == "bf16":
        tol = tol + 2.0 ** -11 * S + 2.0 ** -8 * ref.abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k,n,rank,c0,c1", [
    (1, 32, 1, 0, 0, 1), (1, 4096, 4096, 16, 0, 4096), (3, 96, 33, 2, 0, 33), (8, 1024, 257, 64, 0, 257),
    (9, 64, 256, 0, 0, 256), (128, 512, 700, 5, 100, 600), (257, 2080, 1001, 33, 0, 1001), (300, 1056, 64, 0, 0, 64),
    (515, 4128, 4099, 8, 0, 4099), (1100, 288, 515, 6, 0, 515), (2048, 512, 640, 0, 64, 640), (1057, 96, 65, 64, 0, 65),
    # an odd number of 64-wide stages and several tiles per CTA pair; an adapter on weights taken from planes
    (2000, 4096, 130, 0, 0, 130), (2050, 2592, 264, 20, 0, 264)])
def test_input_gradient(session, cuda, m, k, n, rank, c0, c1, dtype):
    import torch
    packed, scales = _weights(k, n, 7)
    rng = np.random.default_rng(m * n)
    A = (rng.standard_normal((k, max(rank, 1))) * 0.02).astype(np.float32)
    B = (rng.standard_normal((max(rank, 1), n)) * 0.02).astype(np.float32)
    dy = _randn((m, c1 - c0), cuda, 5).to(_dt(dtype))
    dy *= torch.exp2(torch.randint(-12, 3, (m, 1), device=cuda).float()).to(dy.dtype)
    dx = torch.full((m, k), float("nan"), device=cuda, dtype=_dt(dtype))
    with session.weights(packed, scales, k, n, c0, c1) as h:
        if rank:
            h.set_lora(A, B, 2.0 * rank)
        h.input_gradient(dy.data_ptr(), dx.data_ptr(), m, dtype=dtype)
        again = torch.empty_like(dx)
        h.input_gradient(dy.data_ptr(), again.data_ptr(), m, dtype=dtype)
    assert torch.equal(dx, again)
    W, D = _w64(packed, scales, k, n, cuda)[:, c0:c1], dy.double()
    ref, S = D @ W.T, D.abs() @ W.abs().T
    if rank:
        A64, B64 = torch.from_numpy(A).to(cuda).double(), torch.from_numpy(np.ascontiguousarray(B[:, c0:c1])).to(cuda).double()
        ref, S = ref + 2.0 * (D @ B64.T) @ A64.T, S + 2 * 2.0 * (D.abs() @ B64.abs().T) @ A64.abs().T
    _check_dx(dx, dtype, ref, S)
    assert session.device_status(0) == 0


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m", [4, 40])
def test_input_gradient_wide_scales_zero_rows_and_nan(session, cuda, m, dtype):
    """Columns whose scales differ by 2^20, zero rows, zero scales; a row with a NaN and one with an infinity do not
    reach the others."""
    import torch
    k, n = 320, 130
    packed, scales = _weights(k, n, 11)
    scales = np.ascontiguousarray(scales.reshape(n, k // 32)) * np.exp2(np.arange(n) % 21 - 20).astype(np.float32)[:, None]
    scales[5] = 0.0
    dy = _randn((m, n), cuda, 6)
    dy[1] = 0.0
    dy = dy.to(_dt(dtype))
    dx = torch.empty((m, k), device=cuda, dtype=_dt(dtype))
    hurt, out = dy.clone(), torch.empty_like(dx)
    hurt[0, 3], hurt[3, 9] = float("nan"), float("inf")
    with session.weights(packed, scales, k, n) as h:
        h.input_gradient(dy.data_ptr(), dx.data_ptr(), m, dtype=dtype)
        h.input_gradient(hurt.data_ptr(), out.data_ptr(), m, dtype=dtype)
    W = _w64(packed, scales, k, n, cuda)
    _check_dx(dx, dtype, dy.double() @ W.T, dy.double().abs() @ W.abs().T)
    assert not dx[1].any()
    assert not torch.isfinite(out[0]).any() and not torch.isfinite(out[3][W[:, 9] != 0]).any()
    keep = [i for i in range(m) if i not in (0, 3)]
    assert torch.equal(out[keep], dx[keep])


# ------------------------------------------------------------------------------------------------------- cross entropy --
def _loss_ref(x, W, targets, scale):
    import torch
    X = x.double()
    z = X @ W
    S = (X.abs() @ W.abs()).amax(1)
    lse = torch.logsumexp(z, 1)
    used = targets >= 0
    t = targets.clamp(min=0)
    loss = torch.where(used, lse - z.gather(1, t[:, None])[:, 0], 0.0)
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(p).scatter_(1, t[:, None], 1.0)
    g = torch.where(used, scale.double(), 0.0)[:, None]
    return lse, loss, g * ((p - hot) @ W.T), g.abs() * ((p + hot) @ W.abs().T), S


def _check_loss(dtype, got, ref):
    import torch
    (loss, lse, dx), (rl, rloss, rdx, Sdx, S) = got, ref
    dz = 2.0 ** -16 * S
    tol = dz + 2.0 ** -20 * (1 + rl.abs())
    assert ((lse.double() - rl).abs() <= tol).all(), float(((lse.double() - rl).abs() / tol).max())
    assert ((loss.double() - rloss).abs() <= 2 * tol).all(), float(((loss.double() - rloss).abs() / tol).max())
    if dx is not None:
        tol = (2 * dz[:, None] + 2.0 ** -16) * Sdx + 1e-37
        if dtype == "bf16":
            tol = tol + 2.0 ** -10 * Sdx + 2.0 ** -8 * rdx.abs()  # p and W both rounded to f16
        err = (dx.double() - rdx).abs()
        assert torch.isfinite(dx).all() and (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k,n", [(1, 32, 1), (1, 1024, 32003), (5, 64, 259), (8, 2080, 1000), (9, 96, 257),
                                   (130, 512, 512), (257, 1056, 2049), (300, 256, 33000), (1030, 160, 777),
                                   (1025, 32, 5), (2100, 512, 3001), (300, 160, 40000)])
def test_cross_entropy(session, cuda, m, k, n, dtype):
    import torch
    packed, scales = _weights(k, n, 13)
    x = _randn((m, k), cuda, 8).to(_dt(dtype))
    targets = torch.randint(0, n, (m,), device=cuda)
    if m > 4:
        targets[2] = -100
        targets[4] = n - 1
    scale = torch.rand((m,), device=cuda) + 0.5
    loss, lse = torch.full((m,), float("nan"), device=cuda), torch.full((m,), float("nan"), device=cuda)
    dx = torch.full((m, k), float("nan"), device=cuda, dtype=_dt(dtype))
    alone, inplace = torch.empty_like(loss), x.clone()
    with session.weights(packed, scales, k, n) as h:
        h.cross_entropy(x.data_ptr(), targets.data_ptr(), loss.data_ptr(), m, lse=lse.data_ptr(), dx=dx.data_ptr(),
                        row_scale=scale.data_ptr(), dtype=dtype)
        h.cross_entropy(x.data_ptr(), targets.data_ptr(), alone.data_ptr(), m, dtype=dtype)
        l2 = torch.empty_like(loss)
        h.cross_entropy(inplace.data_ptr(), targets.data_ptr(), l2.data_ptr(), m, dx=inplace.data_ptr(),
                        row_scale=scale.data_ptr(), dtype=dtype)
    ref = _loss_ref(x, _w64(packed, scales, k, n, cuda), targets, scale)
    _check_loss(dtype, (loss, lse, dx), ref)
    assert torch.equal(alone, loss) and torch.equal(l2, loss) and torch.equal(inplace, dx)
    if m > 4:
        assert loss[2] == 0 and not dx[2].any()
    assert session.device_status(0) == 0


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m", [6, 70])
def test_cross_entropy_rows_apart(session, cuda, m, dtype):
    """All rows ignored; a row of NaN, a target past the vocabulary, logits far from zero and a row of zeros (uniform)."""
    import torch
    k, n = 128, 700
    packed, scales = _weights(k, n, 17)
    W = _w64(packed, scales, k, n, cuda)
    x = _randn((m, k), cuda, 9)
    x[1] = 0.0
    x[2] *= 400.0
    x = x.to(_dt(dtype))
    targets = torch.randint(0, n, (m,), device=cuda)
    targets[2] = (x[2].double() @ W).argmin()
    one = torch.ones((m,), device=cuda)
    loss, lse, dx = torch.empty((m,), device=cuda), torch.empty((m,), device=cuda), torch.empty_like(x)
    l2, s2, d2 = torch.empty_like(loss), torch.empty_like(lse), torch.empty_like(dx)
    hurt, t2 = x.clone(), targets.clone()
    hurt[4, 7] = float("nan")
    t2[5] = n
    gone = torch.full((m,), -1, device=cuda)
    l3, d3 = torch.empty_like(loss), torch.full_like(dx, float("nan"))
    with session.weights(packed, scales, k, n) as h:
        call = lambda a, t, l, s, d: h.cross_entropy(a.data_ptr(), t.data_ptr(), l.data_ptr(), m, lse=s.data_ptr(),
                                                     dx=d.data_ptr(), dtype=dtype)
        call(x, targets, loss, lse, dx)
        call(hurt, t2, l2, s2, d2)
        call(x, gone, l3, s2.clone(), d3)
    _check_loss(dtype, (loss, lse, dx), _loss_ref(x, W, targets, one))
    assert abs(float(lse[1]) - np.log(n)) <= 2.0 ** -19 * np.log(n)
    assert torch.isnan(l2[4]) and torch.isnan(d2[4]).all() and torch.isnan(s2[4])
    # the target's term is added to the sum of the others, so another target is another order of the same sum: lse
    # within twice its bound, 2^-20 (1 + |lse|), logits being the same
    assert torch.isnan(l2[5]) and torch.isnan(d2[5]).all() and abs(s2[5] - lse[5]) <= 2.0 ** -19 * (1 + abs(lse[5]))
    keep = [i for i in range(m) if i not in (4, 5)]
    assert torch.equal(l2[keep], loss[keep]) and torch.equal(d2[keep], dx[keep])
    assert not l3.any() and not d3.any()


@pytest.mark.parametrize("m", [5, 64])
def test_gradients_against_differences(session, cuda, m):
    """(L(x + h u) - L(x - h u)) / 2h against <dL/dx, u>: the difference is off by h^2/6 |L'''| (third derivatives of a
    log-sum-exp along u are at most 2 max_v |u W_v|^3 ... bounded here by (2 max|uW|)^3) and by 2^-22 |L| / h in fp32."""
    import torch
    k, n, h_ = 256, 500, 2.0 ** -4
    packed, scales = _weights(k, n, 19)
    W = _w64(packed, scales, k, n, cuda)
    x, u = _randn((m, k), cuda, 10), _randn((m, k), cuda, 11)
    u /= (u.double() @ W).abs().amax(1, keepdim=True).float()  # |uW| <= 1
    targets = torch.randint(0, n, (m,), device=cuda)
    out = [torch.empty((m,), device=cuda) for _ in range(3)]
    dx = torch.empty_like(x)
    with session.weights(packed, scales, k, n) as h:
        h.cross_entropy(x.data_ptr(), targets.data_ptr(), out[0].data_ptr(), m, dx=dx.data_ptr())
        for o, v in ((out[1], x + h_ * u), (out[2], x - h_ * u)):
            h.cross_entropy(v.data_ptr(), targets.data_ptr(), o.data_ptr(), m)
    diff = (out[1].double() - out[2].double()) / (2 * h_)
    S = (x.double().abs() @ W.abs()).amax(1)
    tol = h_ ** 2 / 6 * 8 + 2 * (2.0 ** -16 * S + 2.0 ** -20 * (1 + out[0].double())) / h_
    assert ((diff - (dx.double() * u.double()).sum(1)).abs() <= tol).all()


def test_input_gradient_is_the_forward_transposed(session, cuda):
    """<dY, f(x + u) - f(x)> = <dX, u> for the linear layer f with its adapter, f by the fp32 decode path (m <= 8)."""
    import torch
    m, k, n, rank = 4, 512, 320, 8
    packed, scales = _weights(k, n, 23)
    rng = np.random.default_rng(1)
    x, u, dy = _randn((m, k), cuda, 12), _randn((m, k), cuda, 13), _randn((m, n), cuda, 14)
    y0, y1, dx = torch.empty((m, n), device=cuda), torch.empty((m, n), device=cuda), torch.empty((m, k), device=cuda)
    xu = x + u
    with session.weights(packed, scales, k, n) as h:
        h.set_lora(rng.standard_normal((k, rank)).astype(np.float32) * 0.02, rng.standard_normal((rank, n)).astype(np.float32) * 0.02, 16.0)
        h.run(x.data_ptr(), y0.data_ptr(), m)
        h.run(xu.data_ptr(), y1.data_ptr(), m)
        h.input_gradient(dy.data_ptr(), dx.data_ptr(), m)
    a = (dy.double() * (y1.double() - y0.double())).sum(1)
    b = (dx.double() * (xu.double() - x.double())).sum(1)
    W = _w64(packed, scales, k, n, cuda).abs()
    tol = 2.0 ** -13 * (dy.double().abs() * ((x.double().abs() * 2 + u.double().abs()) @ W)).sum(1)  # forward: 1e-4 class
    assert ((a - b).abs() <= tol).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m", [3, 37, 300])
def test_nothing_outside_the_outputs(session, cuda, m, dtype):
    """Buffers that start 16 bytes into an allocation, in front of and behind each a value that has to stay."""
    import torch
    k, n, rank = 352, 130, 5
    packed, scales = _weights(k, n, 41)
    rng = np.random.default_rng(2)

    def room(shape, dt, fill):
        item = torch.empty((), dtype=dt).element_size()
        pad = 16 // item
        buf = torch.full((int(np.prod(shape)) + 2 * pad + 16,), fill, dtype=dt, device=cuda)
        return buf, buf[pad:pad + int(np.prod(shape))].view(shape), pad

    T = _dt(dtype)
    xb, x, _ = room((m, k), T, 7.0)
    yb, dy, _ = room((m, n), T, 7.0)
    x.copy_(_randn((m, k), cuda, 1))
    dy.copy_(_randn((m, n), cuda, 2))
    t = torch.randint(0, n, (m,), device=cuda)
    outs = dict(codes=room((m, k), torch.int8, 55), exps=room((m, k // 32), torch.uint8, 55), back=room((m, k), T, 7.0),
                dx=room((m, k), T, 7.0), dl=room((m, k), T, 7.0), loss=room((m,), torch.float32, 7.0),
                lse=room((m,), torch.float32, 7.0), da=room((k, rank), torch.float32, 7.0), db=room((rank, n), torch.float32, 7.0))
    P = {name: o[1].data_ptr() for name, o in outs.items()}
    with session.weights(packed, scales, k, n) as h, session.weights(packed, scales, k, n) as head:
        h.set_lora(rng.standard_normal((k, rank)).astype(np.float32), rng.standard_normal((rank, n)).astype(np.float32), 3.0)
        session.act8_pack_device(x.data_ptr(), P["codes"], P["exps"], m, k, dtype=dtype)
        session.act8_unpack_device(P["codes"], P["exps"], P["back"], m, k, dtype=dtype)
        h.lora_backward_act8(P["codes"], P["exps"], dy.data_ptr(), m, dtype=dtype, da=P["da"], db=P["db"])
        h.input_gradient(dy.data_ptr(), P["dx"], m, dtype=dtype)
        head.cross_entropy(x.data_ptr(), t.data_ptr(), P["loss"], m, lse=P["lse"], dx=P["dl"], dtype=dtype)
        torch.cuda.synchronize()
    for name, (buf, view, pad) in outs.items():
        keep = buf[0].item()
        assert (buf[:pad] == keep).all() and (buf[pad + view.numel():] == keep).all(), name
        assert (view != keep).any() and torch.isfinite(view.float()).all(), name
    for buf, view, pad in ((xb, x, 16 // x.element_size()), (yb, dy, 16 // x.element_size())):
        assert (buf[:pad] == 7).all() and (buf[pad + view.numel():] == 7).all()


def test_products_keep_to_an_sm_budget(session, cuda):
    """The same results with the handle's launches held to a few SMs."""
    import torch
    m, k, n = 600, 512, 1500
    packed, scales = _weights(k, n, 43)
    dy, x = _randn((m, n), cuda, 3), _randn((m, k), cuda, 4)
    t = torch.randint(0, n, (m,), device=cuda)
    W = _w64(packed, scales, k, n, cuda)
    dx, dl, loss = torch.empty((m, k), device=cuda), torch.empty((m, k), device=cuda), torch.empty((m,), device=cuda)
    with session.weights(packed, scales, k, n) as h:
        for budget in (2, 9, 0):
            h.set_sm_budget(budget)
            h.input_gradient(dy.data_ptr(), dx.data_ptr(), m)
            h.cross_entropy(x.data_ptr(), t.data_ptr(), loss.data_ptr(), m, dx=dl.data_ptr())
            _check_dx(dx, "f32", dy.double() @ W.T, dy.double().abs() @ W.abs().T)
            ref = _loss_ref(x, W, t, torch.ones((m,), device=cuda))
            _check_loss("f32", (loss, ref[0].float(), dl), ref)
    assert session.device_status(0) == 0


def test_two_streams_and_two_graphs_at_once(session, cuda):
    """Calls on two streams of one handle, and two captured graphs of it replayed side by side: no scratch is shared."""
    import torch
    m, k, n = 200, 256, 3000
    packed, scales = _weights(k, n, 47)
    st = [torch.cuda.Stream(cuda) for _ in range(2)]
    xs = [_randn((m, k), cuda, 5 + i) for i in range(2)]
    ts = [torch.randint(0, n, (m,), device=cuda) for _ in range(2)]
    ref, out = [], [[torch.empty((m,), device=cuda), torch.empty((m, k), device=cuda)] for _ in range(2)]
    with session.weights(packed, scales, k, n) as h:
        call = lambda i, s: h.cross_entropy(xs[i].data_ptr(), ts[i].data_ptr(), out[i][0].data_ptr(), m,
                                            dx=out[i][1].data_ptr(), stream=s.cuda_stream)
        for i in range(2):
            call(i, st[0])
            torch.cuda.synchronize()
            ref.append([v.clone() for v in out[i]])
        for _ in range(5):
            for i in range(2):
                call(i, st[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in range(2) for a, b in zip(ref[i], out[i]))
        graphs = []
        for i in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st[i]):
                call(i, st[i])
            graphs.append(g)
        for o in out:
            for v in o:
                v.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(5):
            for i in range(2):
                with torch.cuda.stream(st[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in range(2) for a, b in zip(ref[i], out[i]))
        del graphs
    assert session.device_status(0) == 0


# ------------------------------------------------------------------------------------------------------------ few rows --
# Up to 64 rows have kernels of their own, with fewer than nine from a size on: the bounds above hold for them as they are.
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k,n,rank,c0,c1", [
    (3, 6176, 8003, 2, 0, 8003), (8, 4128, 4099, 0, 0, 4099), (9, 32, 1, 1, 0, 1), (16, 96, 129, 0, 0, 129),
    (17, 160, 1003, 8, 0, 1003), (31, 2080, 515, 0, 0, 515), (32, 4096, 130, 16, 0, 130), (33, 1056, 4099, 64, 0, 4099),
    (63, 288, 77, 0, 0, 77), (64, 512, 2048, 5, 96, 1999), (64, 32, 40003, 3, 0, 40003), (65, 96, 300, 0, 0, 300)])
def test_few_rows_input_gradient(session, cuda, m, k, n, rank, c0, c1, dtype):
    test_input_gradient(session, cuda, m, k, n, rank, c0, c1, dtype)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k,n", [(3, 4096, 12001), (8, 2080, 9001), (9, 32, 1), (16, 288, 129), (17, 96, 40005),
                                   (32, 128, 128), (33, 2080, 1003), (63, 1056, 257), (64, 288, 38500), (65, 64, 130)])
def test_few_rows_cross_entropy(session, cuda, m, k, n, dtype):
    test_cross_entropy(session, cuda, m, k, n, dtype)


@pytest.mark.parametrize("dtype", DT)
def test_few_rows_in_every_setting(session, cuda, dtype):
    """Held to a few SMs, on two streams at once, captured and replayed: the same results; a row of NaN or an ignored one
    changes no other row."""
    import torch
    m, k, n = 40, 416, 5003
    packed, scales = _weights(k, n, 53)
    x, dy = _randn((m, k), cuda, 5).to(_dt(dtype)), _randn((m, n), cuda, 6).to(_dt(dtype))
    t = torch.randint(0, n, (m,), device=cuda)
    W, ones = _w64(packed, scales, k, n, cuda), torch.ones((m,), device=cuda)
    st = [torch.cuda.Stream(cuda) for _ in range(2)]
    new = lambda: [torch.full((m,), float("nan"), device=cuda), torch.full((m,), float("nan"), device=cuda),
                   torch.full((m, k), float("nan"), device=cuda, dtype=x.dtype),
                   torch.full((m, k), float("nan"), device=cuda, dtype=x.dtype)]

    def run(h, o, s, x=x, t=t):
        h.cross_entropy(x.data_ptr(), t.data_ptr(), o[0].data_ptr(), m, lse=o[1].data_ptr(), dx=o[2].data_ptr(),
                        dtype=dtype, stream=s.cuda_stream)
        h.input_gradient(dy.data_ptr(), o[3].data_ptr(), m, dtype=dtype, stream=s.cuda_stream)

    with session.weights(packed, scales, k, n) as h:
        for budget in (2, 7, 0):
            h.set_sm_budget(budget)
            o = new()
            torch.cuda.synchronize()
            run(h, o, st[0])
            torch.cuda.synchronize()
            _check_loss(dtype, (o[0], o[1], o[2]), _loss_ref(x, W, t, ones))
            _check_dx(o[3], dtype, dy.double() @ W.T, dy.double().abs() @ W.abs().T)
        outs = [new(), new()]
        torch.cuda.synchronize()
        for _ in range(5):
            for i in range(2):
                run(h, outs[i], st[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for p in outs for a, b in zip(p, o))
        graphs = []
        for i in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st[i]):
                run(h, outs[i], st[i])
            graphs.append(g)
        for p in outs:
            for v in p:
                v.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(5):
            for i in range(2):
                with torch.cuda.stream(st[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for p in outs for a, b in zip(p, o))
        del graphs
        hurt, ht = x.clone(), t.clone()
        hurt[3, 7], ht[5] = float("nan"), -1
        q = new()
        torch.cuda.synchronize()
        run(h, q, st[0], hurt, ht)
        torch.cuda.synchronize()
        keep = [i for i in range(m) if i not in (3, 5)]
        assert all(torch.equal(a[keep], b[keep]) for a, b in zip(q, o))
        assert torch.isnan(q[0][3]) and torch.isnan(q[2][3]).all() and q[0][5] == 0 and not q[2][5].any()
    assert session.device_status(0) == 0


# ------------------------------------------------------------------------------------------------------------ refusals --
def test_refusals(session, cuda):
    import torch
    k, n, m = 64, 96, 4
    packed, scales = _weights(k, n, 29)
    x = torch.zeros((m + 1, k), device=cuda)
    dy = torch.zeros((m + 1, n), device=cuda)
    t = torch.zeros((m,), dtype=torch.int64, device=cuda)
    loss = torch.zeros((m,), device=cuda)
    codes = torch.zeros((m, k), dtype=torch.int8, device=cuda)
    exps = torch.ones((m, k // 32), dtype=torch.uint8, device=cuda)
    grad, ce, back = (session.raw("spaceslug_q4_weights_" + s) for s in ("input_gradient", "cross_entropy", "lora_backward_act8"))
    with session.weights(packed, scales, k, n) as h:
        w = h.handle
        X, D, T, L, Q, E = (v.data_ptr() for v in (x, dy, t, loss, codes, exps))
        for args in ((None, X, 0, m), (D, None, 0, m), (D, X, 2, m), (D, X, 0, 0), (D + 4, X, 0, m), (D, X + 8, 0, m),
                     (D, X, 0, (1 << 24) + 1)):
            assert grad(w, *args, None) == 1
        for args in ((None, 0, T, None, L, None, None, m), (X, 0, None, None, L, None, None, m), (X, 0, T, None, None, None, None, m),
                     (X, 5, T, None, L, None, None, m), (X, 0, T, None, L, None, None, 0), (X + 4, 0, T, None, L, None, None, m),
                     (X, 0, T, None, L, None, X + 4, m)):
            assert ce(w, *args, None) == 1
        assert back(w, Q, E, D, 0, m, None, None, None) == 1  # no adapter
        h.set_lora(np.zeros((k, 2), np.float32), np.zeros((2, n), np.float32), 2.0)
        assert back(w, None, E, D, 0, m, None, None, None) == 1 and back(w, Q, None, D, 0, m, None, None, None) == 1
        assert back(w, Q, E, None, 0, m, None, None, None) == 1 and back(w, Q, E, D, 3, m, None, None, None) == 1
        assert back(w, Q, E, D, 0, 0, None, None, None) == 1 and back(w, Q + 8, E, D, 0, m, None, None, None) == 1
        assert ce(w, X, 0, T, None, L, None, None, m, None) == 1  # an adapter on the vocabulary
        assert b"adapter" in session._native().spaceslug_last_error()
    assert not torch.cuda.is_current_stream_capturing() and session.device_status(0) == 0


def test_refusals_of_overlap_and_alignment(session, cuda):
    """Buffers that a call writes may share no byte with another (but dx may be x itself), and scalars lie on their own
    size; neighbours are fine."""
    import torch
    k, n, m = 64, 96, 4
    packed, scales = _weights(k, n, 29)
    pool = torch.zeros((1 << 16,), device=cuda)
    P = pool.data_ptr()
    X, D, T, L, E, S = P, P + 4 * m * k, P + 8192, P + 16384, P + 20000, P + 24000
    Q, G, A, B = P + 32768, P + 40000, P + 49152, P + 57344
    grad, ce, back = (session.raw("spaceslug_q4_weights_" + s) for s in ("input_gradient", "cross_entropy", "lora_backward_act8"))

    def clash(code):
        return code == 1 and b"overlaps" in session._native().spaceslug_last_error()

    with session.weights(packed, scales, k, n) as h:
        w = h.handle
        assert grad(w, D, D - 4 * m * k, 0, m, None) == 0  # dx ends where dy begins
        for dx in (D, D - 4 * m * k + 16, D + 4 * m * n - 16):
            assert clash(grad(w, D, dx, 0, m, None))
        good = [X, 0, T, S, L, E, X, m, None]
        assert ce(w, *good) == 0
        for i, v in ((4, X), (4, T), (4, S), (5, L), (5, L + 12), (5, X + 4 * m * k - 4), (6, X + 16), (6, T), (4, T + 8 * m - 4)):
            args = list(good)
            args[i] = v
            assert clash(ce(w, *args)), (i, v)
        for i, v in ((2, T + 4), (3, S + 2), (4, L + 1), (5, E + 2)):
            args = list(good)
            args[i] = v
            assert ce(w, *args) == 1 and b"aligned" in session._native().spaceslug_last_error()
        h.set_lora(np.zeros((k, 2), np.float32), np.zeros((2, n), np.float32), 2.0)
        good = [Q, G, D, 0, m, A, B, None]
        assert back(w, *good) == 0
        for i, v in ((5, D), (5, Q + 16), (5, G), (6, A), (6, A + 4 * (2 * k - 1)), (6, D + 4 * (m * n - 1))):
            args = list(good)
            args[i] = v
            assert clash(back(w, *args)), (i, v)
        for i in (5, 6):
            args = list(good)
            args[i] += 2
            assert back(w, *args) == 1 and b"aligned" in session._native().spaceslug_last_error()
    torch.cuda.synchronize()
    assert session.device_status(0) == 0


# ------------------------------------------------------------------------------------------------------ used together --
def _net(session, k, hidden, vocab, rank, seed):
    rng = np.random.default_rng(seed)
    out = []
    for kk, nn in ((k, hidden), (hidden, k)):
        packed, scales = _weights(kk, nn, seed + kk + nn, 0.01, 0.04)
        A = (rng.standard_normal((kk, rank)) * 0.05).astype(np.float32)
        B = (rng.standard_normal((rank, nn)) * 0.05).astype(np.float32)
        out.append((packed, scales, kk, nn, A, B))
    packed, scales = _weights(k, vocab, seed + 1, 0.01, 0.04)
    return out, (packed, scales, k, vocab)


@pytest.mark.parametrize("m", [6, 200, 2300])
def test_training_step(session, cuda, m):
    """Two int4 layers with adapters under a vocabulary: forward, inputs kept in 8 bits, loss, gradients down to the
    first adapter, on one stream, and once more as a replayed CUDA graph with other inputs."""
    import torch
    k, hidden, vocab, rank = 256, 384, 1000, 8
    layers, head = _net(session, k, hidden, vocab, rank, 31)
    hs = []
    for packed, scales, kk, nn, A, B in layers:
        h = session.weights(packed, scales, kk, nn)
        h.set_lora(A, B, 2.0 * rank)
        hs.append(h)
    hv = session.weights(*head)
    st = torch.cuda.Stream(cuda)
    x = _randn((m, k), cuda, 15)
    t = torch.randint(0, vocab, (m,), device=cuda)
    scale = torch.full((m,), 1.0 / m, device=cuda)
    y1, y2 = torch.empty((m, hidden), device=cuda), torch.empty((m, k), device=cuda)
    c1, e1 = torch.empty((m, k), dtype=torch.int8, device=cuda), torch.empty((m, k // 32), dtype=torch.uint8, device=cuda)
    c2, e2 = torch.empty((m, hidden), dtype=torch.int8, device=cuda), torch.empty((m, hidden // 32), dtype=torch.uint8, device=cuda)
    loss, d2, d1 = torch.empty((m,), device=cuda), torch.empty((m, k), device=cuda), torch.empty((m, hidden), device=cuda)
    g = [(torch.empty((kk, rank), device=cuda), torch.empty((rank, nn), device=cuda)) for _, _, kk, nn, _, _ in layers]

    def step():
        s = st.cuda_stream
        session.act8_pack_device(x.data_ptr(), c1.data_ptr(), e1.data_ptr(), m, k, stream=s)
        hs[0].run(x.data_ptr(), y1.data_ptr(), m, s)
        session.act8_pack_device(y1.data_ptr(), c2.data_ptr(), e2.data_ptr(), m, hidden, stream=s)
        hs[1].run(y1.data_ptr(), y2.data_ptr(), m, s)
        hv.cross_entropy(y2.data_ptr(), t.data_ptr(), loss.data_ptr(), m, dx=d2.data_ptr(), row_scale=scale.data_ptr(), stream=s)
        hs[1].lora_backward_act8(c2.data_ptr(), e2.data_ptr(), d2.data_ptr(), m, da=g[1][0].data_ptr(), db=g[1][1].data_ptr(), stream=s)
        hs[1].input_gradient(d2.data_ptr(), d1.data_ptr(), m, stream=s)
        hs[0].lora_backward_act8(c1.data_ptr(), e1.data_ptr(), d1.data_ptr(), m, da=g[0][0].data_ptr(), db=g[0][1].data_ptr(), stream=s)

    W = [_w64(p, s, kk, nn, cuda) for p, s, kk, nn, _, _ in layers]
    AB = [(torch.from_numpy(A).to(cuda).double(), torch.from_numpy(B).to(cuda).double()) for *_, A, B in layers]
    Wv = _w64(*head, cuda)

    def check():
        torch.cuda.synchronize()
        # what each call got is what the one before gave; 64-bit restatement of each, and of the whole for the loss
        Y1 = x.double() @ W[0] + 2.0 * x.double() @ AB[0][0] @ AB[0][1]
        Y2 = Y1 @ W[1] + 2.0 * Y1 @ AB[1][0] @ AB[1][1]
        assert (y2.double() - Y2).norm() <= 5e-3 * Y2.norm()
        _check_loss("f32", (loss, torch.logsumexp(y2.double() @ Wv, 1).float(), d2), _loss_ref(y2, Wv, t, scale))
        X1 = c1.double() * torch.exp2(e1.double() - 127).repeat_interleave(32, 1)
        X2 = c2.double() * torch.exp2(e2.double() - 127).repeat_interleave(32, 1)
        for X, D, (A, B), (da, db) in ((X2, d2.double(), AB[1], g[1]), (X1, d1.double(), AB[0], g[0])):
            for got, ref in ((da, 2.0 * X.T @ (D @ B.T)), (db, 2.0 * (X @ A).T @ D)):
                assert (got.double() - ref).norm() <= 1e-5 * ref.norm()
        ref = d2.double() @ (W[1] + 2.0 * AB[1][0] @ AB[1][1]).T
        assert (d1.double() - ref).norm() <= 1e-5 * ref.norm()
        # 8-bit copies: half a step of at most 1/127 of a group's largest value per element
        assert ((X2 - y1.double()).abs() <= torch.exp2(e2.double() - 128).repeat_interleave(32, 1)).all()

    with torch.cuda.stream(st):
        step()
        check()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            step()
        x.copy_(_randn((m, k), cuda, 16))
        t.copy_(torch.randint(0, vocab, (m,), device=cuda))
        for v in (loss, d2, d1):
            v.fill_(float("nan"))
        st.synchronize()
        graph.replay()
        check()
        first = [v.clone() for v in (loss, d2, d1, *g[0], *g[1])]
        step()  # an eager step beside the live graph, then the graph again
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, (loss, d2, d1, *g[0], *g[1])))
    del graph
    for h in (*hs, hv):
        h.close()
    assert session.device_status(0) == 0


# --------------------------------------------------------------------------------------- found faults and their mends --
@pytest.mark.parametrize("m", [1, 8, 9, 64, 65, 300, 2100])
def test_logits_of_bf16_rows_at_every_row_count(session, cuda, m):
    """One column and no target: lse is the logit itself.  w = 2^-6 (1 + 2^-12 + 2^-16) is f16 hi + lo without a rest and
    the rows are exact too, so all 2 x 64 products are exact; a sum that cuts each at 2^-24 of S = |z| is off by at most
    2^-17 S, the ways to log2 and back by 2^-21.  (lo and the row in e4m3, 1.0625 each, would be off by 2^-15.)"""
    import torch
    k = 64
    packed = np.full((1, k // 8), 0x11111111, np.uint32)
    scales = np.full((1, k // 32), 2.0 ** -6 * (1 + 2.0 ** -12 + 2.0 ** -16), np.float32)
    x = torch.full((m, k), 1.0625, device=cuda) * torch.exp2(torch.arange(m, device=cuda).float() % 9 - 4)[:, None]
    x = x.bfloat16()
    none, loss = torch.full((m,), -1, dtype=torch.int64, device=cuda), torch.empty((m,), device=cuda)
    lse, dx = torch.empty((m,), device=cuda), torch.empty_like(x)
    z = x.double() @ _w64(packed, scales, k, 1, cuda)[:, 0]
    with session.weights(packed, scales, k, 1) as h:
        for d in (0, dx.data_ptr()):
            h.cross_entropy(x.data_ptr(), none.data_ptr(), loss.data_ptr(), m, lse=lse.data_ptr(), dx=d, dtype="bf16")
            assert ((lse.double() - z).abs() <= 1.0625 * 2.0 ** -17 * z).all(), float(((lse.double() - z).abs() / z).max())
    assert session.device_status(0) == 0


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m", [40, 65, 300, 2050])
@pytest.mark.parametrize("zero", ["all", "one", "one_row"])
def test_input_gradient_with_zero_columns_of_a(session, cuda, m, zero, dtype):
    """Ranks whose column of A is zero (a pruned rank; an adapter that starts from A = 0) add nothing to dX and cost its
    other terms no bits, however large their row of B; one nonzero element makes the column count."""
    import torch
    k, n, rank = 256, 4096, 4
    packed, scales = _weights(k, n, 61, 0.0005, 0.001)
    rng = np.random.default_rng(m)
    A = (rng.standard_normal((k, rank)) * 1e-4).astype(np.float32)
    B = rng.standard_normal((rank, n)).astype(np.float32)
    B[1] *= 1e3
    if zero == "all":
        A[:] = 0.0
    else:
        A[:, 1] = 0.0
        if zero == "one_row":
            A[17, 1] = 1e-6
    dy = _randn((m, n), cuda, 5).to(_dt(dtype))
    dx, bare = (torch.full((m, k), float("nan"), device=cuda, dtype=_dt(dtype)) for _ in range(2))
    with session.weights(packed, scales, k, n) as h:
        h.input_gradient(dy.data_ptr(), bare.data_ptr(), m, dtype=dtype)
        h.set_lora(A, B, 2.0 * rank)
        h.input_gradient(dy.data_ptr(), dx.data_ptr(), m, dtype=dtype)
    W, D = _w64(packed, scales, k, n, cuda), dy.double()
    A64, B64 = torch.from_numpy(A).to(cuda).double(), torch.from_numpy(B).to(cuda).double()
    ref, S = D @ W.T, D.abs() @ W.abs().T
    _check_dx(bare, dtype, ref, S)
    _check_dx(dx, dtype, ref + 2.0 * (D @ B64.T) @ A64.T, S + 2 * 2.0 * (D.abs() @ B64.abs().T) @ A64.abs().T)
    assert session.device_status(0) == 0


@pytest.fixture
def scratch(session):
    hook = session.raw("spaceslug_q4_debug_train_scratch")
    yield lambda rows, weights: hook(rows, weights)
    assert hook(0, 0) == 0


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("weights", [0, 1])  # from 2048 bf16 rows: from planes, and from words
@pytest.mark.parametrize("m,k,n,rank", [(257, 96, 300, 0), (515, 160, 1003, 5), (700, 288, 515, 33), (2100, 416, 130, 16)])
def test_input_gradient_in_blocks_of_rows(session, cuda, scratch, m, k, n, rank, weights, dtype):
    """Blocks of 256 rows and a ragged last one, with the bounds of one block."""
    assert scratch(1, weights) == 0
    test_input_gradient(session, cuda, m, k, n, rank, 0, n, dtype)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("weights", [0, 1])
@pytest.mark.parametrize("m,k,n", [(257, 96, 300), (515, 160, 1003), (700, 288, 257), (2100, 416, 515)])
def test_cross_entropy_in_blocks_of_rows(session, cuda, scratch, m, k, n, weights, dtype):
    """The same for the loss: with lse, row_scale, ignored rows, dx in place of x, and the loss alone."""
    assert scratch(1, weights) == 0
    test_cross_entropy(session, cuda, m, k, n, dtype)


@pytest.mark.parametrize("dtype", DT)
def test_blocks_of_rows_captured_on_two_streams(session, cuda, scratch, dtype):
    """Two graphs of calls in three blocks, replayed side by side: the results of an eager call, which are those of one
    block for the loss (whose logits are not split)."""
    import torch
    m, k, n = 600, 160, 1003
    packed, scales = _weights(k, n, 67)
    x, dy = _randn((m, k), cuda, 5).to(_dt(dtype)), _randn((m, n), cuda, 6).to(_dt(dtype))
    t = torch.randint(0, n, (m,), device=cuda)
    new = lambda: [torch.full((m,), float("nan"), device=cuda), torch.full((m,), float("nan"), device=cuda),
                   torch.full_like(x, float("nan")), torch.full_like(x, float("nan"))]
    st = [torch.cuda.Stream(cuda) for _ in range(2)]
    with session.weights(packed, scales, k, n) as h:
        def run(o, s):
            h.cross_entropy(x.data_ptr(), t.data_ptr(), o[0].data_ptr(), m, lse=o[1].data_ptr(), dx=o[2].data_ptr(),
                            dtype=dtype, stream=s.cuda_stream)
            h.input_gradient(dy.data_ptr(), o[3].data_ptr(), m, dtype=dtype, stream=s.cuda_stream)

        whole, ref, outs = new(), new(), [new(), new()]
        torch.cuda.synchronize()
        run(whole, st[0])
        torch.cuda.synchronize()
        assert scratch(1, 0) == 0
        run(ref, st[0])
        torch.cuda.synchronize()
        assert torch.equal(ref[0], whole[0]) and torch.equal(ref[1], whole[1])
        graphs = []
        for i in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st[i]):
                run(outs[i], st[i])
            graphs.append(g)
        for _ in range(5):
            for i in range(2):
                with torch.cuda.stream(st[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o in outs for a, b in zip(o, ref))
        del graphs
    assert session.device_status(0) == 0


class _KernelNode(ctypes.Structure):  # CUDA_KERNEL_NODE_PARAMS of the driver API
    _fields_ = [("func", ctypes.c_void_p), ("grid", ctypes.c_uint * 3), ("block", ctypes.c_uint * 3),
                ("shared", ctypes.c_uint), ("params", ctypes.c_void_p), ("extra", ctypes.c_void_p),
                ("kern", ctypes.c_void_p), ("ctx", ctypes.c_void_p)]


def _persistent_grids(call, stream):
    """Blocks of the launches that call() makes with more than half an SM's shared memory each, in order of capture."""
    import torch
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g, stream=stream):
        call()
    cu, raw, count, out = ctypes.CDLL("libcuda.so.1"), ctypes.c_void_p(g.raw_cuda_graph()), ctypes.c_size_t(0), []
    assert cu.cuGraphGetNodes(raw, None, ctypes.byref(count)) == 0
    nodes = (ctypes.c_void_p * count.value)()
    assert cu.cuGraphGetNodes(raw, nodes, ctypes.byref(count)) == 0
    for node in nodes:
        kind, p = ctypes.c_int(-1), _KernelNode()
        assert cu.cuGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        if kind.value == 0:
            assert cu.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(node), ctypes.byref(p)) == 0
            if p.shared > 114 * 1024:
                out.append(p.grid[0])
    return out


@pytest.mark.parametrize("dtype,rank", [("f32", 8), ("f32", 33), ("bf16", 8), ("bf16", 64)])
@pytest.mark.parametrize("m", [40, 600])
def test_persistent_launches_keep_to_the_sm_budget(session, cuda, m, dtype, rank):
    """Every launch of a training call that takes an SM's shared memory for itself, the adapter's passes among them, has
    as many blocks as the budget allows at most, and more without one; the results hold their bounds."""
    import torch
    k, n = 1056, 4099
    packed, scales = _weights(k, n, 71)
    rng = np.random.default_rng(3)
    A, B = (rng.standard_normal(s).astype(np.float32) * 0.02 for s in ((k, rank), (rank, n)))
    x, dy = _randn((m, k), cuda, 1), _randn((m, n), cuda, 2).to(_dt(dtype))
    codes, exps, back = _act8(session, x, "f32")
    xs = x.to(dy.dtype)
    t, loss = torch.randint(0, n, (m,), device=cuda), torch.empty((m,), device=cuda)
    dx, dl = torch.empty_like(xs), torch.empty_like(xs)
    da, db = torch.empty((k, rank), device=cuda), torch.empty((rank, n), device=cuda)
    st = torch.cuda.Stream(cuda)
    W, D, A64, B64 = _w64(packed, scales, k, n, cuda), dy.double(), *(torch.from_numpy(v).to(cuda).double() for v in (A, B))
    X = back.double()
    with session.weights(packed, scales, k, n) as h, session.weights(packed, scales, k, n) as head:
        h.set_lora(A, B, 2.0 * rank)
        calls = dict(
            back=lambda s: h.lora_backward_act8(codes.data_ptr(), exps.data_ptr(), dy.data_ptr(), m, dtype=dtype,
                                                da=da.data_ptr(), db=db.data_ptr(), stream=s),
            dx=lambda s: h.input_gradient(dy.data_ptr(), dx.data_ptr(), m, dtype=dtype, stream=s),
            loss=lambda s: head.cross_entropy(xs.data_ptr(), t.data_ptr(), loss.data_ptr(), m, dx=dl.data_ptr(),
                                              dtype=dtype, stream=s))
        for call in calls.values():  # first calls allocate
            call(0)
        torch.cuda.synchronize()
        for name, call in calls.items():
            for budget in (6, 0):
                h.set_sm_budget(budget)
                head.set_sm_budget(budget)
                grids = _persistent_grids(lambda: call(st.cuda_stream), st)
                assert len(grids) >= (1 if name == "dx" else 2), (name, grids)
                if budget:
                    assert max(grids) <= budget, (name, grids)
                else:
                    assert max(grids) > 6, (name, grids)
        h.set_sm_budget(6)
        calls["back"](0)
        calls["dx"](0)
    _check_dx(dx, dtype, D @ W.T + 2.0 * (D @ B64.T) @ A64.T, D.abs() @ W.abs().T + 4.0 * (D.abs() @ B64.abs().T) @ A64.abs().T)
    for got, ref, S in ((da, 2.0 * X.T @ (D @ B64.T), 2.0 * X.abs().T @ (D.abs() @ B64.abs().T)),
                        (db, 2.0 * (X @ A64).T @ D, 2.0 * (X.abs() @ A64.abs()).T @ D.abs())):
        assert ((got.double() - ref).abs() <= 2 * 2.0 ** -16 * S).all()
    assert session.device_status(0) == 0


def test_a_handle_that_only_infers_holds_its_weights_alone(session, cuda):
    """k % 128 != 0: 16 + 4 bytes of words and scales and 4 of exponents per column of 32 k; the training products' padded
    scales (16 more) come with the first call that needs them."""
    import torch
    k, n = 32, 1 << 20
    packed, scales = np.zeros((n, k // 8), np.uint32), np.full((n, 1), 0.01, np.float32)
    session.weights(packed, scales, k, n).close()  # staging buffers
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info(cuda)[0]
    with session.weights(packed, scales, k, n) as h:
        assert free - torch.cuda.mem_get_info(cuda)[0] <= 24 * n + 4 * (2 << 20)  # blocks of 2 MiB
        assert h.n == n


@pytest.mark.parametrize("k", [32, 96, 416])
@pytest.mark.parametrize("first", ["captured", "eager", "two_streams", "two_threads"])
def test_first_training_call_of_a_handle(session, cuda, k, first):
    """The padded scales of a first call: captured (its graph makes its own, and so does a second graph), eager, or from
    two streams or threads at once; the same results each way, and a graph of before works beside the handle's copy."""
    import threading
    import torch
    m, n = 20, 777
    packed, scales = _weights(k, n, 73)
    dy, x = _randn((m, n), cuda, 1), _randn((m, k), cuda, 2)
    t = torch.randint(0, n, (m,), device=cuda)
    W = _w64(packed, scales, k, n, cuda)
    ref = _loss_ref(x, W, t, torch.ones((m,), device=cuda))
    st = [torch.cuda.Stream(cuda) for _ in range(2)]
    new = lambda: [torch.full((m, k), float("nan"), device=cuda), torch.full((m, k), float("nan"), device=cuda),
                   torch.full((m,), float("nan"), device=cuda), torch.full((m,), float("nan"), device=cuda)]
    outs = [new(), new()]
    torch.cuda.synchronize()
    with session.weights(packed, scales, k, n) as h:
        def run(o, s):
            h.input_gradient(dy.data_ptr(), o[0].data_ptr(), m, stream=s.cuda_stream)
            h.cross_entropy(x.data_ptr(), t.data_ptr(), o[2].data_ptr(), m, lse=o[3].data_ptr(), dx=o[1].data_ptr(),
                            stream=s.cuda_stream)

        graphs = []
        if first == "captured":
            for o, s in zip(outs, st):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    run(o, s)
                graphs.append(g)
            for g, s in zip(graphs, st):
                with torch.cuda.stream(s):
                    g.replay()
        elif first == "two_threads":
            threads = [threading.Thread(target=run, args=v) for v in zip(outs, st)]
            for v in threads:
                v.start()
            for v in threads:
                v.join()
        else:
            for o, s in zip(outs, st if first == "two_streams" else st[:1] * 2):
                run(o, s)
        torch.cuda.synchronize()
        after = new()
        run(after, st[0])
        for g, s in zip(graphs, st):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o in (*outs, after):
            _check_dx(o[0], "f32", dy.double() @ W.T, dy.double().abs() @ W.abs().T)
            _check_loss("f32", (o[2], o[3], o[1]), ref)
            assert all(torch.equal(a, b) for a, b in zip(o, after))
        del graphs
    assert session.device_status(0) == 0


# One to eight rows run on either of two sets of kernels, by type, rows, size and adapter: sizes on both sides of the rules.
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k,n,rank", [
    (1, 1056, 8003, 3), (2, 1056, 8003, 0), (3, 1056, 8003, 0), (8, 2080, 2051, 16), (8, 2080, 2051, 0), (5, 4128, 4099, 16),
    (7, 4128, 4099, 64), (2, 4128, 11011, 0), (4, 4128, 12003, 0), (1, 32, 3, 2), (8, 96, 70001, 0)])
def test_one_to_eight_rows_input_gradient(session, cuda, m, k, n, rank, dtype):
    test_input_gradient(session, cuda, m, k, n, rank, 0, n, dtype)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k,n", [(1, 1056, 32003), (1, 2080, 32003), (2, 1056, 32003), (8, 4128, 4099), (8, 1056, 4736),
                                   (8, 1056, 4737), (6, 1056, 8003), (1, 32, 70001), (8, 32, 300001)])
def test_one_to_eight_rows_cross_entropy(session, cuda, m, k, n, dtype):
    test_cross_entropy(session, cuda, m, k, n, dtype)


def _linear_with_adapter(m):
    """Inputs whose adapter weighs more than the weights."""
    k, n, rank = 512, 320, 8
    rng = np.random.default_rng(97 + m)
    A, B, u, dy = ((rng.standard_normal(s) * f).astype(np.float32) for s, f in
                   (((k, rank), 0.2), ((rank, n), 0.2), ((m, k), 1.0), ((m, n), 1.0)))
    return k, n, rank, A, B, u, dy


@pytest.mark.parametrize("m", [4, 40, 300])
def test_input_gradient_is_the_transpose_of_the_layer_with_its_adapter(session, cuda, m):
    """<dY, f(u)> = <dX, u> per row, f by the fp32 decode path in calls of four rows: both sides to 2^-16 of S = sum |dY|
    |u| (|W| + s |A| |B|), and the adapter's part ten times that over the rows."""
    import torch
    k, n, rank, A, B, u, dy = _linear_with_adapter(m)
    packed, scales = _weights(k, n, 23)
    W = _w64(packed, scales, k, n, cuda)
    A64, B64, U, D = (torch.from_numpy(v).to(cuda).double() for v in (A, B, u, dy))
    u, dy = torch.from_numpy(u).to(cuda), torch.from_numpy(dy).to(cuda)
    y, dx = torch.empty((m, n), device=cuda), torch.empty((m, k), device=cuda)
    with session.weights(packed, scales, k, n) as h:
        h.set_lora(A, B, 2.0 * rank)
        for i in range(0, m, 4):
            h.run(u[i:].data_ptr(), y[i:].data_ptr(), 4)
        h.input_gradient(dy.data_ptr(), dx.data_ptr(), m)
    tol = 2 * 2.0 ** -16 * (D.abs() * (U.abs() @ W.abs() + 2 * 2.0 * (U.abs() @ A64.abs()) @ B64.abs())).sum(1)
    adapter = (D * (2.0 * (U @ A64) @ B64)).sum(1).abs()
    assert adapter.norm() >= 10 * tol.norm()
    assert ((D * y.double()).sum(1) - (dx.double() * U).sum(1)).abs().le(tol).all()
    assert session.device_status(0) == 0


@pytest.mark.parametrize("m", [6, 40, 200, 2300])
def test_training_step_in_bf16(session, cuda, m):
    """The step of test_training_step with bf16 activations and gradients between the calls (the forward takes and gives
    fp32: the caller casts), each call against 64 bits, and once more as a replayed graph with other inputs."""
    import torch
    k, hidden, vocab, rank = 256, 384, 1000, 8
    layers, head = _net(session, k, hidden, vocab, rank, 83)
    hs = []
    for packed, scales, kk, nn, A, B in layers:
        h = session.weights(packed, scales, kk, nn)
        h.set_lora(A, B, 2.0 * rank)
        hs.append(h)
    hv = session.weights(*head)
    st, b16 = torch.cuda.Stream(cuda), torch.bfloat16
    x = _randn((m, k), cuda, 15).to(b16)
    t = torch.randint(0, vocab, (m,), device=cuda)
    scale = torch.full((m,), 1.0 / m, device=cuda)
    xf, y1, y2 = torch.empty((m, k), device=cuda), torch.empty((m, hidden), device=cuda), torch.empty((m, k), device=cuda)
    h1, h2 = torch.empty((m, hidden), device=cuda, dtype=b16), torch.empty((m, k), device=cuda, dtype=b16)
    c1, e1 = torch.empty((m, k), dtype=torch.int8, device=cuda), torch.empty((m, k // 32), dtype=torch.uint8, device=cuda)
    c2, e2 = torch.empty((m, hidden), dtype=torch.int8, device=cuda), torch.empty((m, hidden // 32), dtype=torch.uint8, device=cuda)
    loss, lse = torch.empty((m,), device=cuda), torch.empty((m,), device=cuda)
    d2, d1 = torch.empty((m, k), device=cuda, dtype=b16), torch.empty((m, hidden), device=cuda, dtype=b16)
    g = [(torch.empty((kk, rank), device=cuda), torch.empty((rank, nn), device=cuda)) for _, _, kk, nn, _, _ in layers]

    def step():
        s = st.cuda_stream
        session.act8_pack_device(x.data_ptr(), c1.data_ptr(), e1.data_ptr(), m, k, dtype="bf16", stream=s)
        xf.copy_(x)
        hs[0].run(xf.data_ptr(), y1.data_ptr(), m, s)
        h1.copy_(y1)
        session.act8_pack_device(h1.data_ptr(), c2.data_ptr(), e2.data_ptr(), m, hidden, dtype="bf16", stream=s)
        hs[1].run(y1.data_ptr(), y2.data_ptr(), m, s)
        h2.copy_(y2)
        hv.cross_entropy(h2.data_ptr(), t.data_ptr(), loss.data_ptr(), m, lse=lse.data_ptr(), dx=d2.data_ptr(),
                         row_scale=scale.data_ptr(), dtype="bf16", stream=s)
        hs[1].lora_backward_act8(c2.data_ptr(), e2.data_ptr(), d2.data_ptr(), m, dtype="bf16", da=g[1][0].data_ptr(),
                                 db=g[1][1].data_ptr(), stream=s)
        hs[1].input_gradient(d2.data_ptr(), d1.data_ptr(), m, dtype="bf16", stream=s)
        hs[0].lora_backward_act8(c1.data_ptr(), e1.data_ptr(), d1.data_ptr(), m, dtype="bf16", da=g[0][0].data_ptr(),
                                 db=g[0][1].data_ptr(), stream=s)

    W = [_w64(p, s, kk, nn, cuda) for p, s, kk, nn, _, _ in layers]
    AB = [(torch.from_numpy(A).to(cuda).double(), torch.from_numpy(B).to(cuda).double()) for *_, A, B in layers]
    Wv = _w64(*head, cuda)

    def check():
        torch.cuda.synchronize()
        rl, rloss, rdx, Sdx, S = _loss_ref(h2, Wv, t, scale)
        _check_loss("bf16", (loss, lse, None), (rl, rloss, rdx, Sdx, S))
        # As _check_loss, and what f16 leaves of a p far below its tile's largest: 2^14 p / max p is kept in steps of 2^-24
        # at least, so p is off by 2^-25 / 2^14 = 2^-39 of that largest, which is at most 1.  With logits as far apart as
        # these (loss 30 and more) it shows where neither the likely token's nor the target's weight is nonzero.
        tol = (2 * 2.0 ** -16 * S[:, None] + 2.0 ** -16 + 2.0 ** -10) * Sdx + 2.0 ** -8 * rdx.abs() + 1e-37
        tol += 2.0 ** -39 * scale[:, None].double() * Wv.abs().sum(1)
        assert ((d2.double() - rdx).abs() <= tol).all(), float(((d2.double() - rdx).abs() / tol).max())
        X1 = c1.double() * torch.exp2(e1.double() - 127).repeat_interleave(32, 1)
        X2 = c2.double() * torch.exp2(e2.double() - 127).repeat_interleave(32, 1)
        for X, D, (A, B), (da, db) in ((X2, d2.double(), AB[1], g[1]), (X1, d1.double(), AB[0], g[0])):
            for got, ref, S in ((da, 2.0 * X.T @ (D @ B.T), 2.0 * X.abs().T @ (D.abs() @ B.abs().T)),
                                (db, 2.0 * (X @ A).T @ D, 2.0 * (X.abs() @ A.abs()).T @ D.abs())):
                assert ((got.double() - ref).abs() <= 2 * 2.0 ** -16 * S).all()
        D, (A, B) = d2.double(), AB[1]
        _check_dx(d1, "bf16", D @ W[1].T + 2.0 * (D @ B.T) @ A.T, D.abs() @ W[1].abs().T + 4.0 * (D.abs() @ B.abs().T) @ A.abs().T)
        # 8-bit copies: half a step per element
        assert ((X2 - h1.double()).abs() <= torch.exp2(e2.double() - 128).repeat_interleave(32, 1)).all()

    with torch.cuda.stream(st):
        step()
        check()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            step()
        x.copy_(_randn((m, k), cuda, 16))
        t.copy_(torch.randint(0, vocab, (m,), device=cuda))
        for v in (loss, lse, d2, d1):
            v.fill_(float("nan"))
        st.synchronize()
        graph.replay()
        check()
    del graph
    for h in (*hs, hv):
        h.close()
    assert session.device_status(0) == 0


# --------------------------------------------------------------------------------------- calls at the documented edges --
def test_act8_edges_in_bf16(session, cuda):
    """The edges of test_act8_edges that bf16 has, with step bytes that begin at an odd address."""
    import torch
    rows = np.zeros((9, 64), np.float32)
    rows[0, :3] = 127.0, -127.0, 0.5
    rows[1, :3] = 127.5, 1.0, 3.0
    rows[2, :2] = 3.3895313892515355e38, 1.0  # the largest bf16
    rows[3, :2] = 2.0 ** -126, -(2.0 ** -133)
    rows[4, 1], rows[4, 40] = np.inf, 3.0
    rows[5, 33], rows[5, 2] = np.nan, -5.0
    rows[6, :4] = 64.0, 63.5, 62.5, -61.5
    rows[7, :] = -0.0
    rows[8, :] = 2.0 ** 100
    x = torch.from_numpy(rows).to(cuda).bfloat16()
    codes = torch.full((9, 64), 77, dtype=torch.int8, device=cuda)
    room, back = torch.full((1 + 18 + 5,), 99, dtype=torch.uint8, device=cuda), torch.empty_like(x)
    session.act8_pack_device(x.data_ptr(), codes.data_ptr(), room.data_ptr() + 1, 9, 64, dtype="bf16")
    session.act8_unpack_device(codes.data_ptr(), room.data_ptr() + 1, back.data_ptr(), 9, 64, dtype="bf16")
    c, e = _act8_oracle(x.float().cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), c) and np.array_equal(room[1:19].cpu().numpy().reshape(9, 2), e)
    assert room[0] == 99 and (room[19:] == 99).all()
    bad = np.repeat(e == 255, 32, 1)
    b = back.double().cpu().numpy()
    assert bad.sum() == 2 * 32 and np.isnan(b[bad]).all()
    assert np.array_equal(b[~bad], (c * np.exp2(e.astype(np.float64) - 127).repeat(32, 1))[~bad])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m", [5, 40, 300])
def test_cross_entropy_targets_at_the_ends_of_int64(session, cuda, m, dtype):
    """The least int64 takes a row out, the greatest (and one that is the column count past 2^32) is past the columns."""
    import torch
    k, n = 64, 300
    packed, scales = _weights(k, n, 89)
    x = _randn((m, k), cuda, 1).to(_dt(dtype))
    t = torch.randint(0, n, (m,), device=cuda)
    t[1], t[3], t[4] = -2 ** 63, 2 ** 63 - 1, 2 ** 32 + 7
    loss, lse, dx = torch.empty((m,), device=cuda), torch.empty((m,), device=cuda), torch.empty_like(x)
    with session.weights(packed, scales, k, n) as h:
        h.cross_entropy(x.data_ptr(), t.data_ptr(), loss.data_ptr(), m, lse=lse.data_ptr(), dx=dx.data_ptr(), dtype=dtype)
    assert torch.isnan(loss[3:5]).all() and torch.isnan(dx[3:5]).all() and loss[1] == 0 and not dx[1].any()
    keep = torch.tensor([i for i in range(m) if i not in (3, 4)], device=cuda)
    ref = [v[keep] for v in _loss_ref(x, _w64(packed, scales, k, n, cuda), torch.where(t >= n, 0, t), torch.ones((m,), device=cuda))]
    _check_loss(dtype, (loss[keep], lse[keep], dx[keep]), ref)
    assert session.device_status(0) == 0


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m", [3, 40, 300, 2050])
def test_zero_and_negative_scales(session, cuda, m, dtype):
    """A handle of zeros (a uniform softmax, no gradient; dX from the adapter alone) and one with negative scales."""
    import torch
    k, n, rank = 96, 515, 3
    packed, scales = _weights(k, n, 91)
    rng = np.random.default_rng(5)
    A, B = (rng.standard_normal(s).astype(np.float32) * 0.1 for s in ((k, rank), (rank, n)))
    A64, B64 = torch.from_numpy(A).to(cuda).double(), torch.from_numpy(B).to(cuda).double()
    x, dy = _randn((m, k), cuda, 1).to(_dt(dtype)), _randn((m, n), cuda, 2).to(_dt(dtype))
    t, ones = torch.randint(0, n, (m,), device=cuda), torch.ones((m,), device=cuda)
    loss, lse, dl, dx = torch.empty((m,), device=cuda), torch.empty((m,), device=cuda), torch.empty_like(x), torch.empty_like(x)
    signs = np.where(rng.random(scales.shape) < 0.5, -1.0, 1.0).astype(np.float32)
    for sc in (np.zeros_like(scales), scales * signs):
        W = _w64(packed, sc, k, n, cuda)
        with session.weights(packed, sc, k, n) as h:
            h.cross_entropy(x.data_ptr(), t.data_ptr(), loss.data_ptr(), m, lse=lse.data_ptr(), dx=dl.data_ptr(), dtype=dtype)
            h.set_lora(A, B, 2.0 * rank)
            h.input_gradient(dy.data_ptr(), dx.data_ptr(), m, dtype=dtype)
        _check_loss(dtype, (loss, lse, dl), _loss_ref(x, W, t, ones))
        D = dy.double()
        _check_dx(dx, dtype, D @ W.T + 2.0 * (D @ B64.T) @ A64.T, D.abs() @ W.abs().T + 4.0 * (D.abs() @ B64.abs().T) @ A64.abs().T)
        if not sc.any():
            assert not dl.any()
    assert session.device_status(0) == 0


def test_buffers_of_more_than_2_31_elements(session, cuda):
    """70001 rows of 32800 (and 65 of the last rows against 64 bits): bytes and elements past 32 bits in X, its 8-bit form,
    dY and dX of every training call."""
    import torch
    m, wide, few, rank = 70001, 32800, 32, 2
    last = slice(m - 65, m)
    big = torch.empty((m, wide), dtype=torch.bfloat16, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(1)
    for i in range(0, m, 10000):
        big[i:i + 10000] = torch.randn(big[i:i + 10000].shape, device=cuda, generator=gen)
    t = torch.randint(0, few, (m,), device=cuda)
    codes, exps = torch.empty((m, wide), dtype=torch.int8, device=cuda), torch.empty((m, wide // 32), dtype=torch.uint8, device=cuda)
    out = torch.zeros_like(big)
    session.act8_pack_device(big.data_ptr(), codes.data_ptr(), exps.data_ptr(), m, wide, dtype="bf16")
    session.act8_unpack_device(codes.data_ptr(), exps.data_ptr(), out.data_ptr(), m, wide, dtype="bf16")
    c, e = _act8_oracle(big[last].float().cpu().numpy())
    assert np.array_equal(codes[last].cpu().numpy(), c) and np.array_equal(exps[last].cpu().numpy(), e)
    for i in range(0, m, 10000):
        step = torch.exp2(exps[i:i + 10000].float() - 127).repeat_interleave(32, 1)
        assert torch.equal(out[i:i + 10000].float(), codes[i:i + 10000].float() * step)
        assert ((out[i:i + 10000].float() - big[i:i + 10000].float()).abs() <= step / 2).all()
    rng = np.random.default_rng(3)
    # X wide: the adapter's gradients (every row counts) and the loss
    packed, scales = _weights(wide, few, 93)
    A, B = (rng.standard_normal(s).astype(np.float32) * 0.02 for s in ((wide, rank), (rank, few)))
    dy = _randn((m, few), cuda, 4).bfloat16()
    da, db = torch.empty((wide, rank), device=cuda), torch.empty((rank, few), device=cuda)
    loss, lse = torch.empty((m,), device=cuda), torch.empty((m,), device=cuda)
    with session.weights(packed, scales, wide, few) as h:
        h.cross_entropy(big.data_ptr(), t.data_ptr(), loss.data_ptr(), m, lse=lse.data_ptr(), dx=out.data_ptr(), dtype="bf16")
        h.set_lora(A, B, float(rank))
        h.lora_backward_act8(codes.data_ptr(), exps.data_ptr(), dy.data_ptr(), m, dtype="bf16", da=da.data_ptr(), db=db.data_ptr())
    ref = _loss_ref(big[last], _w64(packed, scales, wide, few, cuda), t[last], torch.ones((65,), device=cuda))
    _check_loss("bf16", (loss[last], lse[last], out[last]), ref)
    A64, B64 = torch.from_numpy(A).to(cuda).double(), torch.from_numpy(B).to(cuda).double()
    ra, Sa, rb, Sb = torch.zeros_like(A64), torch.zeros_like(A64), torch.zeros_like(B64), torch.zeros_like(B64)
    for i in range(0, m, 5000):
        X = codes[i:i + 5000].double() * torch.exp2(exps[i:i + 5000].double() - 127).repeat_interleave(32, 1)
        D = dy[i:i + 5000].double()
        ra += X.T @ (D @ B64.T)
        rb += (X @ A64).T @ D
        X.abs_()
        Sa += X.T @ (D.abs() @ B64.abs().T)
        Sb += (X @ A64.abs()).T @ D.abs()
    for got, r, S in ((da, ra, Sa), (db, rb, Sb)):
        assert ((got.double() - r).abs() <= 2 * 2.0 ** -16 * S).all()
    del codes, exps
    # dY wide, in blocks of rows; then dX wide
    packed, scales = _weights(few, wide, 95)
    dx = torch.empty((m, few), dtype=torch.bfloat16, device=cuda)
    with session.weights(packed, scales, few, wide) as h:
        h.input_gradient(big.data_ptr(), dx.data_ptr(), m, dtype="bf16")
    W, D = _w64(packed, scales, few, wide, cuda), big[last].double()
    _check_dx(dx[last], "bf16", D @ W.T, D.abs() @ W.abs().T)
    packed, scales = _weights(wide, few, 93)
    with session.weights(packed, scales, wide, few) as h:
        h.input_gradient(dy.data_ptr(), out.data_ptr(), m, dtype="bf16")
    W, D = _w64(packed, scales, wide, few, cuda), dy[last].double()
    _check_dx(out[last], "bf16", D @ W.T, D.abs() @ W.abs().T)
    assert session.device_status(0) == 0


def test_a_captured_adamw_step_counts_its_replays(session, cuda):
    """Backward and AdamW replayed four times after two eager steps against six eager steps of another handle: the same
    adapter bit for bit, and a first step refused in a capture, which goes on."""
    import torch
    m, k, n, rank = 40, 96, 130, 4
    packed, scales = _weights(k, n, 103)
    rng = np.random.default_rng(4)
    A, B = (rng.standard_normal(s).astype(np.float32) * 0.1 for s in ((k, rank), (rank, n)))
    codes, exps, _ = _act8(session, _randn((m, k), cuda, 1), "f32")
    dy = _randn((m, n), cuda, 2)
    st = torch.cuda.Stream(cuda)
    with session.weights(packed, scales, k, n) as h, session.weights(packed, scales, k, n) as g:
        def step(w, lr=1e-2):
            w.lora_backward_act8(codes.data_ptr(), exps.data_ptr(), dy.data_ptr(), m, stream=st.cuda_stream)
            w.lora_adamw(lr, stream=st.cuda_stream)

        adamw = session.raw("spaceslug_q4_weights_lora_adamw")
        for w in (h, g):
            w.set_lora(A, B, 2.0 * rank)
        torch.cuda.synchronize()
        for _ in range(6):
            step(g)
        h.lora_backward_act8(codes.data_ptr(), exps.data_ptr(), dy.data_ptr(), m, stream=st.cuda_stream)
        first = torch.cuda.CUDAGraph()
        with torch.cuda.graph(first, stream=st):
            dy.mul_(1.0)
            assert adamw(h.handle, 1e-2, 0.9, 0.999, 1e-8, 0.0, st.cuda_stream) == 1
        assert b"before a capture" in session._native().spaceslug_last_error()
        step(h)
        step(h)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            step(h)
        with torch.cuda.stream(st):
            for _ in range(4):
                graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(h.get_lora(rank), g.get_lora(rank)):
            assert a is None or np.array_equal(a, b)
        # six steps of one constant-sign gradient move a parameter by about six rates
        assert np.abs(h.get_lora(rank)[0] - A).max() > 5e-2
        del first, graph
    assert session.device_status(0) == 0
