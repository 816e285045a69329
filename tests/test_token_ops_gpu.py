"""The token-block operators on the GPU against plain 64-bit implementations.

Tolerances.  u(T) is half a step of T relative to the value (bf16 2^-8, f16 2^-11, f32 2^-24); g(n) = n 2^-24 bounds the
relative error of an n-term f32 sum against the sum of the terms' magnitudes.  Where inputs are small integers every
sum is exact in f32 (< 2^24) and the result must equal the correctly rounded one bit for bit: these cases carry the
sizes, layouts and tails; the others carry the arithmetic of the activations."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTS = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F64 = torch.float64


def _ops():
    from svk import ops
    return ops


def _rand(*shape, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dt).cuda()


def _ints(*shape, dt, seed, top=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g).to(dt).cuda()


def _within(got, ref, tol, what=""):
    d = (got.to(F64) - ref).abs()
    bad = ~(d <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d - tol).max()):.3g} over"


# ---------------------------------------------------------------- rotary positions

def _rope_ref(x, pos, freqs, sections, heads, il, inverse):
    """64 bits; and |x| + |y| of every pair, the scale of the f32 arithmetic's error."""
    B, N, C = x.shape
    hd, R = C // heads, sum(sections)
    axis = sum(([a] * n for a, n in enumerate(sections)), [])
    ang = pos.to(F64).expand(B, N, 3)[..., axis] * freqs
    ang = (-ang if inverse else ang)[:, :, None, :]
    y = x.to(F64).view(B, N, heads, hd)
    out, mag = y.clone(), torch.zeros_like(y)
    i = torch.arange(R, device=x.device)
    a, b = (2 * i, 2 * i + 1) if il else (i, i + R)
    p, q = y[..., a], y[..., b]
    out[..., a] = p * ang.cos() - q * ang.sin()
    out[..., b] = p * ang.sin() + q * ang.cos()
    mag[..., a] = mag[..., b] = p.abs() + q.abs()
    return out.view(B, N, C), mag.view(B, N, C)


def _rope_close(got, x, pos, freqs, sections, heads, il, inverse):
    ref, mag = _rope_ref(x, pos, freqs, sections, heads, il, inverse)
    # the reduced angle in f32 (half a turn at most: pi 2^-24 rad), sine and cosine to 4 steps, three f32 roundings
    _within(got, ref, U[x.dtype] * ref.abs() + mag * (math.pi + 4 + 3) * 2.0 ** -24 + 2.0 ** -25, "rope3d")


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("B,N,heads,kv,hd,sections", [
    (1, 1, 1, 1, 6, (1, 1, 1)), (2, 49, 8, 8, 64, (8, 12, 12)), (3, 17, 6, 2, 80, (10, 10, 10)),
    (2, 130, 3, 3, 40, (4, 8, 8)), (1, 2049, 2, 1, 34, (0, 5, 6)), (5, 3, 1, 1, 128, (64, 0, 0)), (1, 7, 2, 2, 18, (3, 3, 3)),
    (2, 40, 4, 4, 72, (7, 6, 6)), (1, 11, 3, 1, 9, (2, 1, 1)), (2, 5, 1, 1, 33, (5, 5, 6)), (1, 300, 5, 5, 7, (1, 1, 1))])
def test_rope3d(cuda, dt, il, B, N, heads, kv, hd, sections):
    ops = _ops()
    q, k = _rand(B, N, heads * hd, dt=dt, seed=1), _rand(B, N, kv * hd, dt=dt, seed=2)
    g = torch.Generator().manual_seed(3)
    pos = torch.randint(-50, 100000, (B, N, 3), generator=g).cuda()
    freqs = ops.rope3d_freqs(sections)
    for p in (pos.int(), pos, pos.float() / 25, pos[0].int()):
        for inverse in (False, True):
            qo, ko = ops.rope3d(q, k, p, freqs, sections, heads, kv, interleaved=il, inverse=inverse)
            _rope_close(qo, q, p, freqs, sections, heads, il, inverse)
            _rope_close(ko, k, p, freqs, sections, kv, il, inverse)


def test_rope3d_is_its_transpose_backwards_and_keeps_the_rest(cuda):
    """<R x, y> = <x, R^T y>: the inverse is the gradient; channels past the pairs are copied bit for bit."""
    ops = _ops()
    B, N, h, hd, sec = 2, 60, 4, 32, (4, 3, 3)
    x, y = _rand(B, N, h * hd, dt=torch.float32, seed=4), _rand(B, N, h * hd, dt=torch.float32, seed=5)
    pos = torch.randint(0, 500, (B, N, 3), generator=torch.Generator().manual_seed(6)).cuda()
    f = ops.rope3d_freqs(sec, shared=True)
    rx, _ = ops.rope3d(x, None, pos, f, sec, h)
    ry, _ = ops.rope3d(y, None, pos, f, sec, h, inverse=True)
    a, b = (rx.to(F64) * y).sum(), (x.to(F64) * ry).sum()
    assert abs(float(a - b)) <= 11 * 2.0 ** -24 * float((x.to(F64).abs() * y.abs()).sum()) * 2
    assert torch.equal(rx.view(B, N, h, hd)[..., 20:], x.view(B, N, h, hd)[..., 20:])
    # against central differences of the loss <R x, y> in one direction
    d = _rand(B, N, h * hd, dt=torch.float32, seed=7)
    up, dn = (ops.rope3d(x + s * d, None, pos, f, sec, h)[0].to(F64) for s in (0.5, -0.5))
    got = (ry.to(F64) * d).sum()
    assert abs(float(((up - dn) * y).sum() - got)) <= 40 * 2.0 ** -24 * float(((x.abs() + d.abs()).to(F64) * y.abs()).sum()) * 2


@pytest.mark.parametrize("dt", DTS)
def test_rope3d_far_positions(cuda, dt):
    """Frame 2^31 - 1 (and 2^40 as int64) at one radian a frame: the angle holds in 64 bits."""
    ops = _ops()
    q = _rand(1, 4, 16, dt=dt, seed=8)
    f = torch.tensor([1.0, 0.7, 1e-3], dtype=F64, device="cuda")
    pos = torch.tensor([[2 ** 31 - 1, 5, 9], [-2 ** 31, 0, 0], [0, 2 ** 30, 1], [123456789, 1, 2 ** 31 - 1]], device="cuda")
    for p in (pos.int(), pos):
        got, _ = ops.rope3d(q, None, p, f, (1, 1, 1), 2)
        # the product pos * f itself is rounded in 64 bits on both sides: 2^31 * 2^-53 rad each
        ref, mag = _rope_ref(q, p, f, (1, 1, 1), 2, False, False)
        _within(got, ref, U[dt] * ref.abs() + mag * (11 * 2.0 ** -24 + 2.0 ** -20), "far")


@pytest.mark.parametrize("dt", DTS)
def test_rope3d_strided_packed_in_place(cuda, dt):
    ops = _ops()
    B, N, h, hd, sec = 3, 21, 4, 32, (6, 5, 5)
    qkv = _rand(B, N, 3 * h * hd, dt=dt, seed=9)
    C = h * hd
    q, k, v = qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:]
    pos = torch.randint(0, 99, (N, 3), generator=torch.Generator().manual_seed(1), dtype=torch.int32).cuda()
    f = ops.rope3d_freqs(sec)
    a, b = ops.rope3d(q, k, pos, f, sec, h)
    keep = v.clone()
    r = ops.rope3d(q, k, pos, f, sec, h, out=(q, k))
    assert r[0] is q and torch.equal(q, a) and torch.equal(k, b) and torch.equal(v, keep)
    x = _rand(B, N, C + 1, dt=dt, seed=10)[..., 1:]               # odd row strides: value by value
    _rope_close(ops.rope3d(x, None, pos, f, sec, h)[0], x, pos, f, sec, h, False, False)
    t = _rand(N, B, C, dt=dt, seed=11).transpose(0, 1)            # time-major
    _rope_close(ops.rope3d(t, None, pos, f, sec, h, interleaved=True)[0], t, pos, f, sec, h, True, False)
    e = _rand(1, N, C, dt=dt, seed=12).expand(B, N, C)            # one input for all batches
    assert torch.equal(ops.rope3d(e, None, pos, f, sec, h)[0], ops.rope3d(e.contiguous(), None, pos, f, sec, h)[0])
    z, _ = ops.rope3d(q[:0], None, pos, f, sec, h)
    assert z.shape == (0, N, C)


@pytest.mark.parametrize("dt", DTS)
def test_rope3d_time_major_in_place(cuda, dt):
    """Tokens outside, batches inside (a stream appends a token of every video): turned in place, packed."""
    ops = _ops()
    B, N, h, hd, sec = 3, 21, 4, 32, (6, 5, 5)
    C = h * hd
    qkv = _rand(N, B, 3 * C, dt=dt, seed=9).transpose(0, 1)
    q, k, v = qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:]
    pos = torch.randint(0, 99, (B, N, 3), generator=torch.Generator().manual_seed(1), dtype=torch.int32).cuda()
    f = ops.rope3d_freqs(sec)
    want, keep = ops.rope3d(q.contiguous(), k.contiguous(), pos, f, sec, h), v.clone()
    out = torch.zeros(N, B, C, device="cuda", dtype=dt).transpose(0, 1)
    assert torch.equal(ops.rope3d(q, None, pos, f, sec, h, out=(out, None))[0], want[0])
    ops.rope3d(q, k, pos, f, sec, h, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, keep)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("hd,sections", [(59, (8, 1, 18)), (24, (3, 3, 3)), (40, (6, 6, 7))])
def test_rope3d_bits_do_not_depend_on_the_piece(cuda, dt, il, hd, sections):
    """A pair is rounded alike wherever it lies in a 16-byte piece: pieces overlap at the end of a part of odd length (both
    write the same bits then, in any order), and in place they do not overlap."""
    ops = _ops()
    B, N, h = 6, 1500, 4
    q = _rand(B, N, h * hd, dt=dt, seed=9)
    pos = torch.randint(0, 5000, (N, 3), generator=torch.Generator().manual_seed(1)).cuda()
    f = ops.rope3d_freqs(sections)
    first = ops.rope3d(q, None, pos, f, sections, h, interleaved=il)[0]
    for _ in range(3):
        assert torch.equal(ops.rope3d(q, None, pos, f, sections, h, interleaved=il)[0], first)
    _rope_close(first, q, pos, f, sections, h, il, False)
    ops.rope3d(q, None, pos, f, sections, h, interleaved=il, out=(q, None))
    assert torch.equal(q, first)


def test_rope3d_positions_that_are_not_finite(cuda):
    ops = _ops()
    q = torch.ones(1, 2, 8, device="cuda")
    pos = torch.tensor([[float("inf"), 1.0, 2.0], [float("nan"), 1.0, 2.0]], device="cuda")
    got, _ = ops.rope3d(q, None, pos, ops.rope3d_freqs((1, 1, 1)), (1, 1, 1), 1, interleaved=True)
    assert bool(got[..., :2].isnan().all()) and bool(got[..., 2:].isfinite().all())


def test_rope3d_refusals(cuda):
    import svk
    ops = _ops()
    q = torch.zeros(2, 5, 32, device="cuda")
    pos = torch.zeros(5, 3, dtype=torch.int32, device="cuda")
    f = ops.rope3d_freqs((2, 3, 3))
    ok = lambda **kw: ops.rope3d(**{**dict(q=q, k=q.clone(), pos=pos, freqs=f, sections=(2, 3, 3), heads=2), **kw})  # noqa: E731
    ok()
    bad = [dict(q=q[0]), dict(heads=3), dict(heads=0), dict(sections=(3, 3, 3)), dict(sections=(-1, 5, 4)), dict(freqs=f[:7]),
           dict(freqs=f.float()), dict(pos=pos[:4]), dict(pos=pos.short()), dict(pos=pos.t().contiguous().t()),
           dict(k=q[:, :4]), dict(k=q.half()), dict(kv_heads=1), dict(q=q.double()), dict(out=(q, None)),
           dict(out=(q.half(), q)), dict(out=(q[:, :4], q)), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)),
           dict(out=(torch.zeros(1, 5, 32, device="cuda").expand(2, 5, 32), torch.zeros_like(q))),
           dict(pos=pos.cpu()), dict(freqs=f.cpu())]
    big = torch.zeros(2, 5, 40, device="cuda")
    bad.append(dict(q=big[..., :32], out=(big[..., 8:], torch.zeros_like(q))))
    same = torch.zeros_like(q)
    bad.append(dict(out=(same, same)))
    for kw in bad:
        with pytest.raises(svk.SvkError):
            ok(**kw)


# ---------------------------------------------------------------- gated feed-forward

def _act64(g, act):
    return {"silu": lambda: g * torch.sigmoid(g), "gelu": lambda: g * torch.special.ndtr(g), "relu": lambda: torch.relu(g)}[act]()


def _dact64(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return s * (1 + g * (1 - s))
    if act == "gelu":
        return torch.special.ndtr(g) + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    return (g > 0).to(F64)


SHAPES = [(1, 8, 8), (1, 1, 1), (7, 33, 50), (16, 64, 72), (17, 40, 512), (32, 100, 333), (33, 96, 64), (64, 17, 129),
          (65, 130, 128), (200, 853, 320), (1000, 96, 61), (129, 256, 1024), (257, 384, 200), (2048, 128, 40)]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("M,H,K", SHAPES)
def test_gated_ffn_exact(cuda, dt, M, H, K):
    """Integers: projections and products exact in f32, so h and the kept projections are the rounded exact values."""
    ops = _ops()
    x, w = _ints(M, K, dt=dt, seed=1), _ints(2 * H, K, dt=dt, seed=2)
    bias = _ints(2 * H, dt=torch.float32, seed=3, top=3)
    for b in (None, bias):
        pre = x.to(F64) @ w.to(F64).t() + (0 if b is None else b.to(F64))
        ref = torch.relu(pre[:, :H]) * pre[:, H:]
        assert float(ref.abs().max()) < 2 ** 24
        h, kept = ops.gated_ffn(x, w, b, act="relu", save=True)
        assert torch.equal(h, ref.to(torch.float32).to(dt)) and torch.equal(kept, pre.to(torch.float32).to(dt))
        assert torch.equal(ops.gated_ffn(x, w, b, act="relu"), h)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("M,H,K", SHAPES)
def test_gated_ffn_bwd_exact(cuda, dt, M, H, K):
    """Integers small enough that dP is exact in every type (|dP| <= 4) and all sums are exact in f32."""
    ops = _ops()
    x, w = _ints(M, K, dt=dt, seed=4), _ints(2 * H, K, dt=dt, seed=5)
    pre, dh = _ints(M, 2 * H, dt=dt, seed=6, top=2), _ints(M, H, dt=dt, seed=7, top=2)
    g, u, d = pre[:, :H].to(F64), pre[:, H:].to(F64), dh.to(F64)
    dp = torch.cat([d * u * (g > 0), d * torch.relu(g)], 1)
    want = [(dp @ w.to(F64)).float().to(dt), (dp.t() @ x.to(F64)).float().to(dt), dp.sum(0).float()]
    got = ops.gated_ffn_bwd(x, w, pre, dh, act="relu")
    for a, b, nm in zip(got, want, ("dx", "dw", "db")):
        assert torch.equal(a, b), (nm, int((a != b).sum()), a.numel())
    for skip in range(3):
        part = ops.gated_ffn_bwd(x, w, pre, dh, act="relu", dx=skip != 0, dw=skip != 1, db=skip != 2)
        assert part[skip] is None and all(torch.equal(p, w_) for i, (p, w_) in enumerate(zip(part, want)) if i != skip)


@pytest.mark.parametrize("M,H,K", [(9000, 136, 120), (12000, 31, 72), (300, 2816, 256), (16640, 256, 512), (13000, 640, 264)])
def test_gated_ffn_large_tiles_exact(cuda, M, H, K):
    """The sizes at which the 128 and 256 tiles and the split token axis run, odd ends included."""
    ops = _ops()
    dt = torch.bfloat16
    x, w = _ints(M, K, dt=dt, seed=8), _ints(2 * H, K, dt=dt, seed=9)
    pre = x.to(F64) @ w.to(F64).t()
    h, kept = ops.gated_ffn(x, w, act="relu", save=True)
    assert torch.equal(kept, pre.float().to(dt))
    assert torch.equal(h, (torch.relu(pre[:, :H]) * pre[:, H:]).float().to(dt))
    pre, dh = _ints(M, 2 * H, dt=dt, seed=6, top=2), _ints(M, H, dt=dt, seed=7, top=2)
    g, u, d = pre[:, :H].to(F64), pre[:, H:].to(F64), dh.to(F64)
    dp = torch.cat([d * u * (g > 0), d * torch.relu(g)], 1)
    dx, dw, db = ops.gated_ffn_bwd(x, w, pre, dh, act="relu")
    assert torch.equal(dx, (dp @ w.to(F64)).float().to(dt))
    assert torch.equal(dw, (dp.t() @ x.to(F64)).float().to(dt))
    assert torch.equal(db, dp.sum(0).float())


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("M,H,K", [(1, 48, 64), (20, 30, 41), (100, 72, 96)])
def test_gated_ffn_values(cuda, dt, act, M, H, K):
    ops = _ops()
    x, w = _rand(M, K, dt=dt, seed=1, scale=2.0), _rand(2 * H, K, dt=dt, seed=2, scale=K ** -0.5)
    b = _rand(2 * H, dt=torch.float32, seed=3)
    X, W = x.to(F64), w.to(F64)
    pre = X @ W.t() + b.to(F64)
    e = (K + 2) * 2.0 ** -24 * (X.abs() @ W.abs().t() + b.to(F64).abs())           # error of a projection
    g, u, eg, eu = pre[:, :H], pre[:, H:], e[:, :H], e[:, H:]
    ref = _act64(g, act) * u
    # |act'| <= 1.13; the activation itself to 2^-21 of |g| (short forms of exp and erf: 1.5e-7 absolute in Phi)
    tol = 1.2 * eg * (u.abs() + eu) + _act64(g, act).abs() * eu + g.abs() * u.abs() * 2.0 ** -21
    got, kept = ops.gated_ffn(x, w, b, act=act, save=True)
    _within(got, ref, U[dt] * (ref.abs() + tol) + tol + 2.0 ** -25, "h")
    _within(kept, pre, U[dt] * (pre.abs() + e) + e + 2.0 ** -25, "pre")


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_ffn_bwd_values(cuda, dt, act):
    ops = _ops()
    M, H, K = 75, 40, 56
    x, w = _rand(M, K, dt=dt, seed=1), _rand(2 * H, K, dt=dt, seed=2, scale=K ** -0.5)
    pre, dh = _rand(M, 2 * H, dt=dt, seed=3, scale=2.0), _rand(M, H, dt=dt, seed=4)
    P = pre.to(F64).requires_grad_()
    (_act64(P[:, :H], act) * P[:, H:]).backward(dh.to(F64))
    dp = P.grad
    g, u, d = pre[:, :H].to(F64), pre[:, H:].to(F64), dh.to(F64)
    # dP in f32: factors to 2^-21 of |dh u| (1 + |g|) and |dh g|; rounded once (half a step, or half the smallest f16 step)
    e32 = torch.cat([d.abs() * u.abs() * (1 + g.abs()), d.abs() * g.abs()], 1) * 2.0 ** -21
    e = e32 + U[dt] * (dp.abs() + e32) + (2.0 ** -25 if dt == torch.float16 else 0)
    dx, dw, db = ops.gated_ffn_bwd(x, w, pre, dh, act=act)
    X, W = x.to(F64), w.to(F64)
    for got, ref, tol in ((dx, dp @ W, (e + (2 * H) * 2.0 ** -24 * (dp.abs() + e)) @ W.abs()),
                          (dw, dp.t() @ X, (e + M * 2.0 ** -24 * (dp.abs() + e)).t() @ X.abs()),
                          (db, dp.sum(0), (e32 + M * 2.0 ** -24 * (dp.abs() + e32)).sum(0))):
        u_ = U[got.dtype]
        _within(got, ref, tol + u_ * (ref.abs() + tol) + 2.0 ** -25, act)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_ffn_bwd_kept_gates_that_left_the_range(cuda, dt, act):
    """Gates kept as infinities: act and act' are 0 below, act' is 1 above; integers elsewhere, so all of it is exact."""
    ops = _ops()
    M, H, K = 3, 24, 16
    x, w = _ints(M, K, dt=dt, seed=1), _ints(2 * H, K, dt=dt, seed=2)
    dh, u = _ints(M, H, dt=dt, seed=3, top=3), _ints(M, H, dt=dt, seed=4, top=3)
    g = torch.full((M, H), -float("inf"), device="cuda", dtype=dt)
    pre = torch.cat([g, u], 1)
    dx, dw, db = ops.gated_ffn_bwd(x, w, pre, dh, act=act)
    assert not bool(dx.any()) and not bool(dw.any()) and not bool(db.any())       # NaN.any() is true
    dx, dw, db = ops.gated_ffn_bwd(x, w, torch.cat([-g, u], 1), dh, act=act)
    assert torch.equal(db[:H].to(F64), (dh.to(F64) * u.to(F64)).sum(0))
    assert torch.equal(dw[:H].to(F64), (dh.to(F64) * u.to(F64)).t() @ x.to(F64))


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_ffn_bwd_kept_projections_that_left_the_range_behind_zeros(cuda, dt, act):
    """Projections kept as infinities (f16's range) where the other factor is zero: the forward pass held them in f32
    and gave 0, so does the gradient.  All of it is exact."""
    ops = _ops()
    inf = float("inf")
    M, H, K = 3, 24, 16
    x, w = _ints(M, K, dt=dt, seed=1), _ints(2 * H, K, dt=dt, seed=2)
    dh = _ints(M, H, dt=dt, seed=3, top=3)
    big = torch.full((M, H), inf, device="cuda", dtype=dt)
    big[:, ::2] = -inf
    shut = torch.full((M, H), -1e4, device="cuda", dtype=dt)           # act and act' are zeros of f32
    none = torch.zeros(M, H, device="cuda", dtype=dt)
    for pre, d in ((torch.cat([shut, big], 1), dh), (torch.cat([big, big], 1), none), (torch.cat([big.abs(), big], 1), none)):
        for t in ops.gated_ffn_bwd(x, w, pre, d, act=act):
            assert not bool(t.any())                                   # NaN.any() is true
    # open gates: the infinities pass where dh is not zero, and nowhere else
    one = torch.ones(1, K, device="cuda", dtype=dt)
    d = dh[:1]
    dx, dw, db = ops.gated_ffn_bwd(one, w, torch.cat([big[:1].abs(), big[:1].abs()], 1), d, act=act)
    want = torch.where(d[0] == 0, 0.0, d[0].float() * inf)
    assert torch.equal(db, torch.cat([want, want])) and torch.equal(dw.float(), db[:, None].expand(2 * H, K))
    # NaN is never hidden, nor an infinite dh
    nan = torch.full((1, H), float("nan"), device="cuda", dtype=dt)
    for g, u, d in ((shut[:1], nan, none[:1]), (nan, shut[:1], none[:1]), (shut[:1], shut[:1], big[:1])):
        assert bool(ops.gated_ffn_bwd(one, w, torch.cat([g, u], 1), d, act=act)[0].isnan().all())


def test_gated_ffn_bwd_products_past_the_range_behind_closed_gates(cuda):
    """dh * u leaves f32's range, act' is zero: the gradient of the gate is zero."""
    ops = _ops()
    for dt in (torch.float32, torch.bfloat16):
        x, w = _ints(2, 16, dt=dt, seed=1), _ints(16, 16, dt=dt, seed=2)
        pre = torch.full((2, 16), 2.0 ** 100, device="cuda", dtype=dt)
        pre[:, :8] = -1e4
        for act in ("silu", "gelu", "relu"):
            for t in ops.gated_ffn_bwd(x, w, pre, pre[:, 8:].contiguous(), act=act):
                assert not bool(t.any())


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("M,H,K", [(1, 1, 1), (7, 33, 50), (200, 853, 320), (1000, 96, 61), (4874, 33, 1043), (16640, 256, 512),
                                   (833, 2505, 803), (325, 4734, 1797), (4357, 365, 650)])
def test_gated_ffn_bwd_added_to_gradient_buffers(cuda, dt, M, H, K):
    """dw and db added to f32 buffers, in f32: the sums (to 4 M) are exact, whatever the type would round them to.  What
    lies around the buffers stays."""
    ops = _ops()
    x, w = _ints(M, K, dt=dt, seed=4), _ints(2 * H, K, dt=dt, seed=5)
    pre, dh = _ints(M, 2 * H, dt=dt, seed=6, top=2), _ints(M, H, dt=dt, seed=7, top=2)
    g, u, d = pre[:, :H].to(F64), pre[:, H:].to(F64), dh.to(F64)
    dp = torch.cat([d * u * (g > 0), d * torch.relu(g)], 1)
    dw, db = dp.t().contiguous() @ x.to(F64), dp.sum(0)
    n = 2 * H * K
    flat = torch.full((n + 2 * H + 12,), 5.0, device="cuda")                 # a flat buffer of gradients, at an odd place
    gw, gb = flat[3:3 + n].view(2 * H, K), flat[3 + n + 4:3 + n + 4 + 2 * H]
    start = _ints(2 * H, K, dt=torch.float32, seed=8, top=9000)
    gw.copy_(start)
    gb.copy_(start[:, 0])
    for turn in (1, 2):
        dx, rw, rb = ops.gated_ffn_bwd(x, w, pre, dh, act="relu", dw=gw, db=gb)
        assert rw is gw and rb is gb
        assert torch.equal(gw.to(F64), start.to(F64) + turn * dw) and torch.equal(gb.to(F64), start[:, 0].to(F64) + turn * db)
        assert torch.equal(dx, (dp @ w.to(F64)).float().to(dt))
    assert bool((flat[:3] == 5).all()) and bool((flat[3 + n:3 + n + 4] == 5).all()) and bool((flat[3 + n + 4 + 2 * H:] == 5).all())
    # one of them added to, the other written
    gb.zero_()
    _, w16, rb = ops.gated_ffn_bwd(x, w, pre, dh, act="relu", dx=False, db=gb)
    assert rb is gb and torch.equal(gb.to(F64), db) and w16.dtype == dt and torch.equal(w16, dw.float().to(dt))
    gw.zero_()
    _, rw, rb = ops.gated_ffn_bwd(x, w, pre, dh, act="relu", dw=gw)
    assert torch.equal(gw.to(F64), dw) and torch.equal(rb.to(F64), db)
    # no tokens: nothing is added
    ops.gated_ffn_bwd(x[:0], w, pre[:0], dh[:0], act="relu", dw=gw, db=gb)
    assert torch.equal(gw.to(F64), dw) and torch.equal(gb.to(F64), db)


def test_gated_ffn_bwd_entry_adds_nothing_without_tokens(cuda):
    from svk import _lib
    lib = _lib.load()
    x, w = torch.zeros(1, 16, device="cuda"), torch.zeros(24, 16, device="cuda")
    dw, db = torch.ones(24, 16, device="cuda"), torch.ones(24, device="cuda")
    p, st = x.data_ptr(), torch.cuda.current_stream().cuda_stream
    for add, left in ((3, (1, 1)), (1, (1, 0)), (2, (0, 1))):
        dw.fill_(1)
        db.fill_(1)
        assert lib.svk_gated_ffn_bwd_add(0, p, 16, w.data_ptr(), 16, p, p, 12, p, 16, dw.data_ptr(), db.data_ptr(), add, 0, 12,
                                         16, 0, None, 0, st) == 0
        torch.cuda.synchronize()
        assert bool((dw == left[0]).all()) and bool((db == left[1]).all())


def test_gated_ffn_bwd_added_to_buffers_in_a_graph(cuda):
    """Captured: every replay adds once more; eager calls between them too."""
    ops = _ops()
    M, H, K, dt = 3000, 40, 72, torch.bfloat16
    x, w = _ints(M, K, dt=dt, seed=4), _ints(2 * H, K, dt=dt, seed=5)
    pre, dh = _ints(M, 2 * H, dt=dt, seed=6, top=2), _ints(M, H, dt=dt, seed=7, top=2)
    _, one, oneb = ops.gated_ffn_bwd(x.float(), w.float(), pre.float(), dh.float(), act="relu")
    gw, gb = torch.zeros(2 * H, K, device="cuda"), torch.zeros(2 * H, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.gated_ffn_bwd(x, w, pre, dh, act="relu", dw=gw, db=gb)
    n = 0
    for _ in range(3):
        g.replay()
        ops.gated_ffn_bwd(x, w, pre, dh, act="relu", dx=False, dw=gw, db=gb)
        n += 2
        torch.cuda.synchronize()
        assert torch.equal(gw, n * one) and torch.equal(gb, n * oneb)


def test_gated_ffn_gradient_against_differences(cuda):
    """f32: the derivative of sum(h * dh) along random directions of x, w and the bias, by central differences of the
    forward kernel.  Steps of 2^-6: third-order term ~ 2^-12 of the slope's scale, rounding ~ 2^-24 / 2^-6."""
    ops = _ops()
    M, H, K, s = 50, 24, 32, 2.0 ** -6
    dt = torch.float32
    x, w = _rand(M, K, dt=dt, seed=1), _rand(2 * H, K, dt=dt, seed=2, scale=K ** -0.5)
    b, dh = _rand(2 * H, dt=dt, seed=3), _rand(M, H, dt=dt, seed=4)
    for act in ("silu", "gelu"):
        _, pre = ops.gated_ffn(x, w, b, act=act, save=True)
        grads = ops.gated_ffn_bwd(x, w, pre, dh, act=act)
        loss = lambda x_, w_, b_: float((ops.gated_ffn(x_, w_, b_, act=act).to(F64) * dh.to(F64)).sum())  # noqa: E731
        for i, t in enumerate((x, w, b)):
            d = _rand(*t.shape, dt=dt, seed=10 + i, scale=1.0 if i == 0 else K ** -0.5)
            up, dn = [x, w, b], [x, w, b]
            up[i], dn[i] = t + s * d, t - s * d
            slope = (loss(*up) - loss(*dn)) / (2 * s)
            want = float((grads[i].to(F64) * d.to(F64)).sum())
            scale = float((grads[i].to(F64).abs() * d.to(F64).abs()).sum())
            assert abs(slope - want) <= 2.0 ** -10 * scale, (act, i, slope, want, scale)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("M", [3, 40])
def test_gated_ffn_views(cuda, dt, M):
    """Column ranges of wider buffers, misaligned rows, the newest token of a batch, a given output; what lies around
    the output is left as it was."""
    ops = _ops()
    H, K = 24, 40
    wide, wbuf = _ints(M, K + 24, dt=dt, seed=1), _ints(2 * H, K + 9, dt=dt, seed=2)
    ref = lambda x, w: (lambda p: torch.relu(p[..., :H]) * p[..., H:])(x.to(F64) @ w.to(F64).t()).float().to(dt)  # noqa: E731
    for x in (wide[:, 8:8 + K], wide[:, 1:1 + K]):
        for w in (wbuf[:, :K].contiguous(), wbuf[:, 3:3 + K]):
            out = torch.full((M + 2, H + 5), 7.0, device="cuda", dtype=dt)
            ops.gated_ffn(x, w, act="relu", out=out[1:-1, 2:2 + H])
            assert torch.equal(out[1:-1, 2:2 + H], ref(x, w))
            out[1:-1, 2:2 + H] = 7.0
            assert bool((out == 7.0).all())
    seq = _ints(M, 6, K, dt=dt, seed=3)
    w = wbuf[:, :K].contiguous()
    assert torch.equal(ops.gated_ffn(seq[:, -1:], w, act="relu"), ref(seq[:, -1:], w))
    pre, dh = _ints(M, 2 * H, dt=dt, seed=6, top=2), _ints(M, H + 3, dt=dt, seed=7, top=2)[:, 3:]
    for x, w in ((wide[:, 8:8 + K], w), (wide[:, 1:1 + K], wbuf[:, 3:3 + K])):
        for a, b in zip(ops.gated_ffn_bwd(x, w, pre, dh, act="relu"),
                        ops.gated_ffn_bwd(x.contiguous(), w.contiguous(), pre, dh.contiguous(), act="relu")):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dt", DTS)
def test_gated_ffn_no_tokens(cuda, dt):
    ops = _ops()
    x, w = torch.empty(0, 16, device="cuda", dtype=dt), _rand(24, 16, dt=dt, seed=1)
    h, pre = ops.gated_ffn(x, w, save=True)
    assert h.shape == (0, 12) and pre.shape == (0, 24)
    dx, dw, db = ops.gated_ffn_bwd(x, w, pre, h)
    assert dx.shape == (0, 16) and not bool(dw.any()) and not bool(db.any()) and dw.dtype == dt


def test_gated_ffn_bwd_entry_without_tokens(cuda):
    """The C entry itself: sums over no tokens are zeros, written to dW and db."""
    from svk import _lib
    lib = _lib.load()
    x, w = torch.zeros(1, 16, device="cuda"), torch.zeros(24, 16, device="cuda")
    dw, db = torch.ones(24, 16, device="cuda"), torch.ones(24, device="cuda")
    p = x.data_ptr()
    rc = lib.svk_gated_ffn_bwd(0, p, 16, w.data_ptr(), 16, p, p, 12, p, 16, dw.data_ptr(), db.data_ptr(), 0, 12, 16, 0, None,
                               0, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0 and not bool(dw.any()) and not bool(db.any())


@pytest.mark.parametrize("M", [5, 100])
def test_gated_ffn_not_finite_stays_in_its_row(cuda, M):
    """A token that holds an infinity or a NaN spoils its own row only (also the rows that share its tile)."""
    ops = _ops()
    x, w = _rand(M, 64, dt=torch.bfloat16, seed=1), _rand(48, 64, dt=torch.bfloat16, seed=2)
    clean = ops.gated_ffn(x, w)
    x2 = x.clone()
    x2[2, 5], x2[4, 63] = float("nan"), float("inf")
    got = ops.gated_ffn(x2, w)
    rest = [i for i in range(M) if i not in (2, 4)]
    assert torch.equal(got[rest], clean[rest]) and bool(got[2].isnan().all()) and not bool(got[4].isfinite().all())


def test_gated_ffn_refusals(cuda):
    import svk
    ops = _ops()
    x, w = torch.zeros(6, 16, device="cuda"), torch.zeros(8, 16, device="cuda")
    b, pre, dh = torch.zeros(8, device="cuda"), torch.zeros(6, 8, device="cuda"), torch.zeros(6, 4, device="cuda")
    f = lambda **kw: ops.gated_ffn(**{**dict(x=x, w=w, bias=b), **kw})  # noqa: E731
    g = lambda **kw: ops.gated_ffn_bwd(**{**dict(x=x, w=w, pre=pre, dh=dh), **kw})  # noqa: E731
    f(); g()
    for kw in (dict(w=w[:7]), dict(w=w[:, :15]), dict(w=w.half()), dict(x=x.double()), dict(x=x.t()), dict(bias=b[:7]),
               dict(bias=b.half()), dict(act="tanh"), dict(act=None), dict(out=x[:, :4]), dict(out=dh.half()), dict(out=dh[:5]),
               dict(w=w[:0]), dict(x=x[:, :0]), dict(out=torch.zeros(1, 4, device="cuda").expand(6, 4)), dict(w=w.cpu()),
               dict(x=x.cpu()), dict(bias=b.cpu()), dict(w=torch.zeros(16, 8, device="cuda").t())):
        with pytest.raises(svk.SvkError):
            f(**kw)
    for kw in (dict(pre=pre[:, :7]), dict(pre=pre[:5]), dict(dh=dh[:5]), dict(dh=dh[:, :3]), dict(pre=pre.half()), dict(dh=dh.half()),
               dict(pre=torch.zeros(6, 9, device="cuda")[:, :8]), dict(act="none"), dict(w=w[:7]), dict(dh=dh.cpu())):
        with pytest.raises(svk.SvkError):
            g(**kw)


# ---------------------------------------------------------------- 8-bit integer products

_127TH = torch.tensor(1 / 127, dtype=torch.float32)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("M,K", [(1, 1), (5, 7), (3, 64), (130, 333), (9, 512), (4, 520), (2, 1024), (3, 2048), (2, 4096), (2, 5000), (2, 4099)])
def test_quant_rows(cuda, dt, M, K):
    """The scale is one f32 product and x / scale an f32 division, correctly rounded on both sides: equal bit for bit."""
    ops = _ops()
    x = _rand(M, K, dt=dt, seed=1, scale=3.0)
    if M > 1:
        x[1] = 0
    q, s = ops.quant_rows(x)
    xf = x.float().cpu()
    want_s = xf.abs().amax(1) * _127TH
    want_q = torch.where(want_s[:, None] > 0, torch.round(xf / want_s[:, None]), torch.zeros_like(xf))
    assert q.shape == (M, K) and s.shape == (M,) and q.stride(0) % 16 == 0
    assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu(), want_q.to(torch.int8))
    # a row's values are kept to half a step of its scale
    _within(q.to(F64) * s.to(F64)[:, None], x.to(F64), (0.5 + 2.0 ** -15) * s.to(F64)[:, None].expand(M, K) + 1e-30, "values")


@pytest.mark.parametrize("dt", DTS)
def test_quant_rows_has_the_codes_of_the_torch_expression(cuda, dt):
    ops = _ops()
    x = _rand(2000, 1056, dt=dt, seed=7)
    s = x.float().abs().amax(1) / 127
    q, sc = ops.quant_rows(x)
    assert torch.equal(sc, s) and torch.equal(q.float(), torch.round(x.float() / s[:, None]))


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("K", [17, 333, 512, 1000])
def test_quant_rows_of_many_short_rows(cuda, dt, K):
    """One row a wave or several: the same bits."""
    ops = _ops()
    x = _rand(7003, K, dt=dt, seed=3)
    q, s = ops.quant_rows(x)
    xf = x.float().cpu()
    want = xf.abs().amax(1) * _127TH
    assert torch.equal(s.cpu(), want) and torch.equal(q.cpu(), torch.round(xf / want[:, None]).to(torch.int8))
    few = ops.quant_rows(x[-600:])
    assert torch.equal(q[-600:], few[0]) and torch.equal(s[-600:], few[1])


def test_quant_rows_more_rows_than_one_launch(cuda):
    """2^26 rows, 64 threads each, are 2^32 threads."""
    ops = _ops()
    M = (1 << 26) + 5
    x = torch.zeros(M, 4, device="cuda", dtype=torch.float16)
    at = torch.tensor([0, 1, (1 << 25) - 1, 1 << 25, (1 << 26) - 1, 1 << 26, M - 1], device="cuda")
    x[at] = _ints(len(at), 4, dt=torch.float16, seed=1, top=9)
    q, s = ops.quant_rows(x)
    q2, s2 = ops.quant_rows(x[at])
    assert torch.equal(q[at], q2) and torch.equal(s[at], s2) and int((s != 0).sum()) == int((s2 != 0).sum())


def test_quant_rows_ties_and_scales_of_all_sizes(cuda):
    """Quotients on and next to half integers (16-bit values divide to exact ties often), and scales from subnormal to
    1e36: still the correctly rounded quotient, rounded."""
    ops = _ops()
    n = torch.arange(-127, 128, dtype=torch.float32) * 0.5
    x = torch.cat([n, torch.nextafter(n, n + 1), torch.nextafter(n, n - 1), torch.tensor([127.0, 126.99999])])
    g = torch.Generator().manual_seed(5)
    rows = [x * 2.0 ** e * f for e in (-140, -126, -100, -60, 0, 60, 110) for f in (1.0, 1.1, 1.9999999)]
    rows += [torch.randn(len(x), generator=g).half().float() * 2.0 ** -e for e in range(12)]
    x = torch.stack(rows)
    s = x.abs().amax(1, keepdim=True) * _127TH
    want = torch.where(s > 0, torch.round(x / s), torch.zeros_like(x)).clamp(-127, 127)
    q, sc = ops.quant_rows(x.cuda())
    fine = s[:, 0] >= 2.0 ** -126                 # a subnormal scale is a rough number, but the same on both sides
    assert torch.equal(sc.cpu()[fine], s[fine, 0]) and torch.equal(q.cpu()[fine].float(), want[fine])
    assert int(q.abs().max()) <= 127
    for dt in (torch.float16, torch.bfloat16):
        y = (torch.randint(-2000, 2001, (500, 256), generator=g).float() / 64).to(dt)
        s = y.float().abs().amax(1, keepdim=True) * _127TH
        assert torch.equal(ops.quant_rows(y.cuda())[0].cpu().float(), torch.round(y.float() / s))


def test_quant_rows_not_finite_tiny_and_views(cuda):
    ops = _ops()
    x = _rand(6, 40, dt=torch.float32, seed=2)
    x[1, 3], x[2, 39], x[3, 0] = float("inf"), float("nan"), -float("inf")
    x[4] *= 1e-40                                          # subnormal values: the scale may round to few bits or to zero
    q, s = ops.quant_rows(x)
    assert bool(s[1:4].isnan().all()) and not bool(q[1:4].any()) and bool(s[[0, 4, 5]].isfinite().all())
    assert int(q.abs().max()) <= 127
    b = _rand(4, 3, 50, dt=torch.bfloat16, seed=3)
    for v in (b[:, -1:], b[:, 0, :24], b[..., 1:1 + 24]):
        q, s = ops.quant_rows(v)
        q2, s2 = ops.quant_rows(v.contiguous())
        assert q.shape == v.shape and s.shape == v.shape[:-1] and torch.equal(q, q2) and torch.equal(s, s2)
    q, s = ops.quant_rows(b[:0])
    assert q.shape == (0, 3, 50) and s.shape == (0, 3)


def _codes(M, K, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8).cuda()


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 100, 64), (16, 33, 130), (17, 64, 1000), (32, 7, 47), (33, 65, 128), (100, 130, 61),
                                   (257, 129, 512), (1000, 640, 144), (300, 20, 4096)])
def test_gemm_i8(cuda, dt, M, N, K):
    ops = _ops()
    a, w = _codes(M, K, 1), _codes(N, K, 2)
    sa, sw = _rand(M, dt=torch.float32, seed=3).abs() / 64, _rand(N, dt=torch.float32, seed=4).abs() / 64
    b, r = _rand(N, dt=torch.float32, seed=5), _rand(M, N, dt=dt, seed=6)
    acc = (a.cpu().to(torch.int64) @ w.cpu().to(torch.int64).t()).cuda().to(F64)
    for act, bias, res in ((None, None, None), ("gelu", b, None), ("relu", b, r), ("tanh", None, r)):
        y = acc * sa.to(F64)[:, None] * sw.to(F64)
        z = y if bias is None else y + bias.to(F64)
        v = {None: z, "gelu": z * torch.special.ndtr(z), "relu": torch.relu(z), "tanh": torch.tanh(z)}[act]
        ref = v if res is None else v + res.to(F64)
        # the integer to f32, two products, the bias: 4 roundings; activations to 2^-21 of the argument; the residual's sum
        tol = 1.2 * 4 * 2.0 ** -24 * (y.abs() + (0 if bias is None else bias.to(F64).abs())) + z.abs() * 2.0 ** -21
        tol = tol + 2.0 ** -24 * (ref.abs() + v.abs())
        got = ops.gemm_i8(a, sa, w, sw, bias, act=act, residual=res, dtype=dt)
        assert got.dtype == dt
        _within(got, ref, U[dt] * (ref.abs() + tol) + tol + 2.0 ** -25, f"{act}")


@pytest.mark.parametrize("M,N,K", [(4100, 1032, 160), (5000, 3000, 96), (13000, 264, 48)])
def test_gemm_i8_large_tiles_exact(cuda, M, N, K):
    ops = _ops()
    a, w = _codes(M, K, 1), _codes(N, K, 2)
    one = lambda n: torch.ones(n, device="cuda")  # noqa: E731
    got = ops.gemm_i8(a, one(M), w, one(N), dtype=torch.float32)
    assert torch.equal(got.to(F64), a.to(F64) @ w.to(F64).t())      # < 2^24: exact in f32


def test_gemm_i8_exact_sums_views_and_extremes(cuda):
    ops = _ops()
    one = lambda n: torch.ones(n, device="cuda")  # noqa: E731
    for M in (2, 70):
        # the longest reduction at the largest codes: 131071 * 128 * 128 = 2^31 - 2^14 in int32
        a = torch.full((M, 131071), -128, dtype=torch.int8, device="cuda")
        w = torch.full((3, 131071), -128, dtype=torch.int8, device="cuda")
        w[1] = 127
        got = ops.gemm_i8(a, one(M), w, one(3), dtype=torch.float32)
        want = torch.tensor([128.0 * 128 * 131071, -128.0 * 127 * 131071, 128.0 * 128 * 131071], device="cuda")
        assert torch.equal(got, want.expand(M, 3))
        ab, wb = _codes(M, 90, 3), _codes(20, 90, 4)
        for x, y in ((ab[:, 16:80], wb[:, 16:80]), (ab[:, 1:60], wb[:, 2:61])):
            out = torch.full((M + 2, 26), 9.0, device="cuda")
            ops.gemm_i8(x, one(M), y, one(20), out=out[1:-1, 3:23])
            assert torch.equal(out[1:-1, 3:23].to(F64), x.to(F64) @ y.to(F64).t())
            out[1:-1, 3:23] = 9.0
            assert bool((out == 9.0).all())
        # out is the residual
        r = _ints(M, 20, dt=torch.float32, seed=1, top=9)
        want = r + ops.gemm_i8(ab, one(M), wb, one(20), dtype=torch.float32)
        ops.gemm_i8(ab, one(M), wb, one(20), residual=r, out=r)
        assert torch.equal(r, want)
        # a row whose scale is NaN spoils its own outputs only
        s = one(M)
        s[1] = float("nan")
        y = ops.gemm_i8(ab, s, wb, one(20), dtype=torch.float32)
        assert bool(y[1].isnan().all()) and bool(y[0].isfinite().all())
    e = ops.gemm_i8(_codes(4, 16, 1)[:0], one(0), _codes(5, 16, 2), one(5))
    assert e.shape == (0, 5) and e.dtype == torch.float16


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("act", [None, "relu", "gelu", "tanh"])
@pytest.mark.parametrize("M", [5, 100])
def test_gemm_i8_not_finite_tokens_are_nan_behind_every_activation(cuda, dt, act, M):
    ops = _ops()
    x, w = _rand(M, 64, dt=torch.float32, seed=1), ops.quant_rows(_rand(48, 64, dt=torch.float32, seed=2))
    clean = ops.gemm_i8(*ops.quant_rows(x), *w, act=act, dtype=dt)
    x[2, 7], x[4, 0] = float("inf"), float("nan")
    got = ops.gemm_i8(*ops.quant_rows(x), *w, act=act, dtype=dt)
    rest = [i for i in range(M) if i not in (2, 4)]
    assert torch.equal(got[rest], clean[rest]) and bool(got[[2, 4]].isnan().all())


@pytest.mark.parametrize("K", [61, 333, 1001])
def test_gemm_i8_tokens_that_end_inside_a_chunk(cuda, K):
    """Codes of quant_rows keep whatever their buffer held behind a row of K % 16 values; it must not be seen."""
    ops = _ops()
    M, N = 100, 72
    buf = torch.full((M, (K + 15) // 16 * 16), 77, dtype=torch.int8, device="cuda")
    a, w = buf[:, :K], _codes(N, K, 2)
    a.copy_(_codes(M, K, 1))
    one = lambda n: torch.ones(n, device="cuda")  # noqa: E731
    want = a.to(F64) @ w.to(F64).t()
    assert torch.equal(ops.gemm_i8(a, one(M), w, one(N), dtype=torch.float32).to(F64), want)
    wb = torch.full((N, (K + 15) // 16 * 16), -55, dtype=torch.int8, device="cuda")
    wb[:, :K] = w
    assert torch.equal(ops.gemm_i8(a, one(M), wb[:, :K], one(N), dtype=torch.float32).to(F64), want)
    assert torch.equal(ops.gemm_i8(a[:5], one(5), wb[:, :K], one(N), dtype=torch.float32).to(F64), want[:5])


def test_i8_refusals(cuda):
    import svk
    ops = _ops()
    a, w = _codes(4, 16, 1), _codes(6, 16, 2)
    sa, sw = torch.ones(4, device="cuda"), torch.ones(6, device="cuda")
    r = torch.zeros(4, 6, device="cuda", dtype=torch.float16)
    f = lambda **kw: ops.gemm_i8(**{**dict(a=a, a_scale=sa, w=w, w_scale=sw), **kw})  # noqa: E731
    f()
    for kw in (dict(a=a.float()), dict(w=w.short()), dict(w=w[:, :15]), dict(a_scale=sa[:3]), dict(w_scale=sw[:5]),
               dict(a_scale=sa.half()), dict(bias=sw[:5]), dict(residual=r[:3]), dict(residual=r.float()), dict(act="silu"),
               dict(dtype=torch.float64), dict(dtype=torch.int8), dict(out=r[:3]), dict(a=a.t()), dict(w=w[:0]), dict(w=w.cpu()),
               dict(out=r.double()), dict(w_scale=torch.ones(12, device="cuda")[::2]), dict(a=a.cpu()),
               dict(a=torch.zeros(2, 131072, dtype=torch.int8, device="cuda"), a_scale=sa[:2],
                    w=torch.zeros(6, 131072, dtype=torch.int8, device="cuda")),
               dict(out=torch.zeros(1, 6, device="cuda").expand(4, 6)), dict(residual=r, out=r.flatten()[:24].view(6, 4).t())):
        with pytest.raises(svk.SvkError):
            f(**kw)
    for bad in (a, torch.zeros(3, 0, device="cuda"), torch.zeros(3, 4, device="cuda").t(), torch.zeros(3, 4, dtype=F64, device="cuda")):
        with pytest.raises(svk.SvkError):
            ops.quant_rows(bad)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [40, 4000])
def test_gelu_of_16_bit_results_down_its_tail(cuda, dt, M):
    """GELU(g) alone (up = 1), as gated_ffn and gemm_i8 form it.  erfc is off by 1.5e-7 at most, so the result by
    0.75e-7 |g|, and six f32 roundings of a correction of at most |g| / 2; as the correction is a positive multiple of
    exp(-g^2 / 2) that tends to 0.7779 / 0.5642 of the true one, the tail is within 0.4 of itself as well.  Then half a
    step (f16: half the smallest one, 2^-25)."""
    ops = _ops()
    g = torch.linspace(-12, 9, M).to(dt).cuda()
    x, w = torch.ones(M, 8, device="cuda", dtype=dt), torch.zeros(32, 8, device="cuda", dtype=dt)
    x[:, 0] = g
    w[:16, 0] = w[16:, 1] = 1
    h = ops.gated_ffn(x, w, act="gelu")
    G = g.to(F64)
    ref = G * 0.5 * torch.erfc(-G * 0.5 ** 0.5)        # (ndtr cancels in 64 bits: 0 from -8.3 down)
    err = 0.75e-7 * G.abs() + 6 * 2.0 ** -24 * G.abs() / 2 + 2.0 ** -24 * ref.abs()
    err = torch.where(G < -2, torch.minimum(err, 0.4 * ref.abs()), err)
    tol = err + U[dt] * (ref.abs() + err) + (2.0 ** -25 if dt == torch.float16 else 2.0 ** -134)
    _within(h, ref[:, None].expand(M, 16), tol[:, None].expand(M, 16), "gated")
    # 8-bit: codes times scales that give the same arguments (one product of powers of two, so exact)
    a = torch.ones(M, 16, device="cuda", dtype=torch.int8)
    one = torch.ones(16, 16, device="cuda", dtype=torch.int8)
    y = ops.gemm_i8(a, g.float() / 16, one, torch.ones(16, device="cuda"), act="gelu", dtype=dt)
    _within(y, ref[:, None].expand(M, 16), tol[:, None].expand(M, 16), "i8")


# ---------------------------------------------------------------- every tile size, split and second launch

_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _plan(entry, *args):
    """(tile side, reduction split, tile side of the rows behind) that the library takes for these sizes."""
    import ctypes
    from svk import _lib
    out = (ctypes.c_long * 4)()
    _lib.call(entry, *args, out)
    return out[0], out[1] > 1, out[3]


F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
# tokens, hidden, K, (tile side, tile side of the last rows); rows of results of whole 64-byte lines and of any length
_FWD16 = [(196, 4240, 152, (128, 0)), (16396, 35, 156, (128, 0)), (5124, 392, 848, (128, 64)), (2566, 787, 835, (128, 64)),
          (24910, 208, 152, (256, 0)), (24910, 224, 152, (256, 0)), (26051, 198, 154, (256, 0)), (22730, 332, 150, (256, 64)), (19628, 400, 322, (256, 128)),
          (18545, 516, 258, (256, 128))]
_FWD32 = [(24790, 40, 82, (128, 0)), (26594, 35, 76, (128, 0)), (33632, 162, 82, (128, 64)), (28379, 200, 80, (256, 0)), (28379, 208, 80, (256, 0)),
          (28213, 194, 75, (256, 0)), (34747, 196, 77, (256, 64)), (16426, 516, 77, (256, 128))]


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dt,M,H,K,tiles", [(F32, *c) for c in _FWD32] + [(d, *c) for d in (BF16, F16) for c in _FWD16])
def test_gated_ffn_every_tile(cuda, dt, M, H, K, tiles, act):
    """With biases and kept projections; ReLU exact on integers, the others within test_gated_ffn_values' bounds."""
    ops = _ops()
    side, split, rest = _plan("svk_gated_ffn_plan", _CODE[dt], 0, M, H, K)
    assert (side, rest) == tiles and not split
    if act == "relu":
        x, w, b = _ints(M, K, dt=dt, seed=1), _ints(2 * H, K, dt=dt, seed=2), _ints(2 * H, dt=F32, seed=3, top=3)
        pre = x.to(F64) @ w.to(F64).t() + b.to(F64)
        got, kept = ops.gated_ffn(x, w, b, act=act, save=True)
        assert torch.equal(kept, pre.float().to(dt)) and torch.equal(got, (torch.relu(pre[:, :H]) * pre[:, H:]).float().to(dt))
        return
    x, w = _rand(M, K, dt=dt, seed=1, scale=2.0), _rand(2 * H, K, dt=dt, seed=2, scale=K ** -0.5)
    b = _rand(2 * H, dt=F32, seed=3)
    X, W = x.to(F64), w.to(F64)
    pre = X @ W.t() + b.to(F64)
    e = (K + 2) * 2.0 ** -24 * (X.abs() @ W.abs().t() + b.to(F64).abs())
    g, u, eg, eu = pre[:, :H], pre[:, H:], e[:, :H], e[:, H:]
    ref = _act64(g, act) * u
    tol = 1.2 * eg * (u.abs() + eu) + _act64(g, act).abs() * eu + g.abs() * u.abs() * 2.0 ** -21
    got, kept = ops.gated_ffn(x, w, b, act=act, save=True)
    _within(got, ref, U[dt] * (ref.abs() + tol) + tol + 2.0 ** -25, "h")
    _within(kept, pre, U[dt] * (pre.abs() + e) + e + 2.0 ** -25, "pre")


# product (1: dx, 2: dW), tokens, hidden, K, (tile side, split, tile side of the last rows)
_BWD16 = [(1, 10982, 80, 136, (128, False, 0)), (1, 3301, 420, 1235, (128, False, 64)), (1, 513, 4531, 67, (128, True, 0)),
          (1, 24757, 80, 408, (256, False, 0)), (1, 24757, 80, 416, (256, False, 0)), (1, 16698, 75, 652, (256, False, 0)), (1, 33473, 82, 385, (256, False, 64)),
          (1, 33155, 130, 544, (256, False, 128)), (1, 4370, 2674, 195, (256, True, 0)), (2, 155, 4208, 200, (128, False, 0)),
          (2, 833, 2505, 803, (128, False, 64)), (2, 4874, 33, 1043, (128, True, 0)), (2, 156, 4108, 1415, (256, False, 0)),
          (2, 164, 4676, 1674, (256, False, 64)), (2, 325, 4734, 1797, (256, False, 128)), (2, 325, 4734, 1792, (256, False, 64)), (2, 5378, 2056, 200, (256, True, 0))]
_BWD32 = [(1, 26259, 38, 66, (128, False, 0)), (1, 33398, 39, 327, (128, False, 64)), (1, 4133, 517, 66, (128, True, 0)),
          (1, 6344, 41, 1930, (256, False, 0)), (1, 15190, 40, 784, (256, False, 0)), (1, 21829, 39, 663, (256, False, 64)), (1, 26475, 40, 642, (256, False, 128)),
          (1, 1489, 1096, 656, (256, True, 0)), (2, 78, 5062, 266, (128, False, 0)), (2, 129, 3910, 1153, (128, False, 64)),
          (2, 1029, 371, 641, (128, True, 0)), (2, 80, 5515, 1102, (256, False, 0)), (2, 80, 5515, 1104, (256, False, 0)), (2, 79, 4785, 1667, (256, False, 64)),
          (2, 77, 5728, 1544, (256, False, 128)), (2, 4413, 1040, 216, (256, True, 0))]


@pytest.mark.parametrize("dt,product,M,H,K,plan", [(F32, *c) for c in _BWD32] + [(d, *c) for d in (BF16, F16) for c in _BWD16])
def test_gated_ffn_bwd_every_tile(cuda, dt, product, M, H, K, plan):
    """Integers as in test_gated_ffn_bwd_exact; the sums stay under 4 * 34000 < 2^24."""
    ops = _ops()
    assert _plan("svk_gated_ffn_plan", _CODE[dt], product, M, H, K) == plan
    x, w = _ints(M, K, dt=dt, seed=4), _ints(2 * H, K, dt=dt, seed=5)
    pre, dh = _ints(M, 2 * H, dt=dt, seed=6, top=2), _ints(M, H, dt=dt, seed=7, top=2)
    g, u, d = pre[:, :H].to(F64), pre[:, H:].to(F64), dh.to(F64)
    dp = torch.cat([d * u * (g > 0), d * torch.relu(g)], 1)
    dx, dw, db = ops.gated_ffn_bwd(x, w, pre, dh, act="relu")
    assert torch.equal(dx, (dp @ w.to(F64)).float().to(dt))
    assert torch.equal(dw, (dp.t().contiguous() @ x.to(F64)).float().to(dt))
    assert torch.equal(db, dp.sum(0).float())


_I8 = [(16416, 74, 315, (128, 0)), (17310, 72, 300, (128, 0)), (33444, 72, 1145, (128, 64)), (25289, 400, 332, (256, 0)), (25289, 416, 332, (256, 0)),
       (25127, 434, 303, (256, 0)), (33836, 388, 309, (256, 64)), (15836, 2128, 307, (256, 128))]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("M,N,K,tiles", _I8)
def test_gemm_i8_every_tile(cuda, dt, M, N, K, tiles):
    """Scales, bias, every activation and a residual that is also the output, within test_gemm_i8's bounds."""
    ops = _ops()
    side, split, rest = _plan("svk_gemm_i8_plan", M, N, K)
    assert (side, rest) == tiles and not split
    a, w = _codes(M, K, 1), _codes(N, K, 2)
    sa, sw = _rand(M, dt=F32, seed=3).abs() / 64, _rand(N, dt=F32, seed=4).abs() / 64
    b, r = _rand(N, dt=F32, seed=5), _rand(M, N, dt=dt, seed=6)
    y = (a.to(F64) @ w.to(F64).t()) * sa.to(F64)[:, None] * sw.to(F64)
    for act, bias, res in ((None, None, None), ("gelu", b, r), ("relu", b, r), ("tanh", b, None), (None, b, r)):
        z = y if bias is None else y + bias.to(F64)
        v = {None: z, "gelu": z * torch.special.ndtr(z), "relu": torch.relu(z), "tanh": torch.tanh(z)}[act]
        ref = v if res is None else v + res.to(F64)
        tol = 1.2 * 4 * 2.0 ** -24 * (y.abs() + (0 if bias is None else bias.to(F64).abs())) + z.abs() * 2.0 ** -21
        tol = tol + 2.0 ** -24 * (ref.abs() + v.abs())
        got = ops.gemm_i8(a, sa, w, sw, bias, act=act, residual=res, dtype=dt)
        _within(got, ref, U[dt] * (ref.abs() + tol) + tol + 2.0 ** -25, f"{act}")
        if res is not None:
            own = res.clone()
            ops.gemm_i8(a, sa, w, sw, bias, act=act, residual=own, out=own)
            assert torch.equal(own, got)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("width", [1500, 3001, 5000, 7003])
@pytest.mark.parametrize("K", [77, 2304])
def test_few_tokens_every_width(cuda, dt, width, K):
    """One to four blocks of weight rows a workgroup, one to four blocks of tokens, rows that end inside a piece and rows
    of several turns of the waves; all exact."""
    ops = _ops()
    w, b = _ints(2 * width, K, dt=dt, seed=2), _ints(2 * width, dt=F32, seed=3, top=3)
    wq, one = _codes(2 * width, K, 4), torch.ones(2 * width, device="cuda")
    for M in (1, 16, 20, 33, 64):
        x = _ints(M, K, dt=dt, seed=M)
        pre = x.to(F64) @ w.to(F64).t() + b.to(F64)
        ref = torch.relu(pre[:, :width]) * pre[:, width:]
        assert float(ref.abs().max()) < 2 ** 24
        h, kept = ops.gated_ffn(x, w, b, act="relu", save=True)
        assert torch.equal(h, ref.float().to(dt)) and torch.equal(kept, pre.float().to(dt))
        a = _codes(M, K, M)
        want = (a.to(F64) @ wq.to(F64).t()).float()
        assert torch.equal(ops.gemm_i8(a, one[:M], wq, one, dtype=F32), want)


# ---------------------------------------------------------------- together

def _block(ops, x, pos, freqs, p, eps=1e-6):
    """A pre-norm transformer block over video tokens; what the backward pass needs."""
    C, h = p["wo"].shape[0], p["heads"]
    xn = ops.layernorm(x, p["g1"], p["b1"], eps)
    qkv = ops.gemm(xn, p["wqkv"])
    q, k, v = qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:]
    ops.rope3d(q, k, pos, freqs, p["sections"], h, out=(q, k))
    a = ops.attention(q, k, v, h, (C // h) ** -0.5)
    y = ops.gemm(a, p["wo"], residual=x)
    yn = ops.layernorm(y, p["g2"], p["b2"], eps)
    hid, pre = ops.gated_ffn(yn, p["wgu"], p["bgu"], save=True)
    return ops.gemm(hid, p["wd"], residual=y), (xn, q, k, v, a, y, yn, hid, pre)


def _block_ref(x, pos, freqs, p, eps=1e-6):
    F = torch.nn.functional
    B, N, C = x.shape
    h = p["heads"]
    xn = F.layer_norm(x, (C,), p["g1"], p["b1"], eps)
    q, k, v = (xn @ p["wqkv"].t()).split(C, -1)
    axis = sum(([i] * n for i, n in enumerate(p["sections"])), [])
    ang = (pos.to(F64)[:, axis] * freqs)[None, :, None]
    R = len(axis)

    def turn(t):
        t = t.reshape(B, N, h, -1)
        a, b, rest = t[..., :R], t[..., R:2 * R], t[..., 2 * R:]
        return torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos(), rest], -1).transpose(1, 2)
    s = turn(q) @ turn(k).transpose(-1, -2) * (C // h) ** -0.5
    a = (s.softmax(-1) @ v.reshape(B, N, h, -1).transpose(1, 2)).transpose(1, 2).reshape(B, N, C)
    y = x + a @ p["wo"].t()
    yn = F.layer_norm(y, (C,), p["g2"], p["b2"], eps)
    g, u = (yn @ p["wgu"].t() + p["bgu"]).chunk(2, -1)
    return y + (g * torch.sigmoid(g) * u) @ p["wd"].t()


def _params(dt, C=64, hid=88, heads=2):
    s = C ** -0.5
    return dict(heads=heads, sections=(4, 5, 5), g1=1 + _rand(C, dt=torch.float32, seed=1, scale=0.1),
                b1=_rand(C, dt=torch.float32, seed=2, scale=0.1), g2=1 + _rand(C, dt=torch.float32, seed=3, scale=0.1),
                b2=_rand(C, dt=torch.float32, seed=4, scale=0.1), wqkv=_rand(3 * C, C, dt=dt, seed=5, scale=s),
                wo=_rand(C, C, dt=dt, seed=6, scale=s), wgu=_rand(2 * hid, C, dt=dt, seed=7, scale=s),
                bgu=_rand(2 * hid, dt=torch.float32, seed=8, scale=0.1), wd=_rand(C, hid, dt=dt, seed=9, scale=hid ** -0.5))


def _grid(t, h, w):
    i = torch.arange(t * h * w, device="cuda")
    return torch.stack([1000 + i // (h * w), i // w % h, i % w], -1).int()


def test_video_block_forward_and_gradients_f32(cuda):
    """One block forward and backward in f32 against 64-bit autograd.  2e-5 of the result's largest value, the f32 bound
    of the kernels it is chained from (test_kernels_gpu.py); gradients pass through twice as many."""
    ops = _ops()
    p, pos = _params(torch.float32), _grid(2, 5, 5)
    x, dz = _rand(3, 50, 64, dt=torch.float32, seed=20), _rand(3, 50, 64, dt=torch.float32, seed=21)
    freqs = ops.rope3d_freqs(p["sections"])
    out, (xn, q, k, v, a, y, yn, hid, pre) = _block(ops, x, pos, freqs, p)
    p64 = {n: t.to(F64).requires_grad_() if torch.is_tensor(t) else t for n, t in p.items()}
    x64 = x.to(F64).requires_grad_()
    ref = _block_ref(x64, pos, freqs, p64)
    ref.backward(dz.to(F64))
    _within(out, ref.detach(), 2e-5 * float(ref.detach().abs().max()), "block")
    # backward, kernel by kernel
    C, h = 64, p["heads"]
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    gw = {n: torch.zeros_like(p[n]) for n in ("wqkv", "wo", "wd", "g1", "b1", "g2", "b2")}
    ops.gemm_wgrad(flat(dz), flat(hid), gw["wd"])
    dhid = ops.gemm(dz, p["wd"].t().contiguous())
    dyn, gw["wgu"], gw["bgu"] = ops.gated_ffn_bwd(yn, p["wgu"], pre, dhid)
    dy = ops.layernorm_bwd(y, dyn, p["g2"], 1e-6, dres=dz, dgamma=gw["g2"], dbeta=gw["b2"])
    ops.gemm_wgrad(flat(dy), flat(a), gw["wo"])
    da = ops.gemm(dy, p["wo"].t().contiguous())
    dq, dk, dv = ops.attention_bwd(q, k, v, a, da, h, (C // h) ** -0.5)
    dq, dk = ops.rope3d(dq, dk, pos, freqs, p["sections"], h, inverse=True)
    dqkv = torch.cat([dq, dk, dv], -1)
    ops.gemm_wgrad(flat(dqkv), flat(xn), gw["wqkv"])
    dx = ops.layernorm_bwd(x, ops.gemm(dqkv, p["wqkv"].t().contiguous()), p["g1"], 1e-6, dres=dy, dgamma=gw["g1"],
                           dbeta=gw["b1"])
    for n, g in dict(gw, x=dx).items():
        r = (x64 if n == "x" else p64[n]).grad
        _within(g, r, 4e-5 * float(r.abs().max()), n)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_video_block_16bit_and_streaming(cuda, dt):
    """The block in 16 bits; and its newest token alone, against the cached keys and values of the clip, as a stream
    runs it.  Errors: about 12 roundings of values of the result's size on either path."""
    ops = _ops()
    p, pos = _params(dt), _grid(2, 5, 5)
    x = _rand(3, 50, 64, dt=dt, seed=20)
    freqs = ops.rope3d_freqs(p["sections"])
    out, (xn, q, k, v, *_) = _block(ops, x, pos, freqs, p)
    ref = _block_ref(x.to(F64), pos, freqs, {n: t.to(F64) if torch.is_tensor(t) else t for n, t in p.items()})
    tol = 12 * U[dt] * float(ref.abs().max())
    _within(out, ref, tol, "block")
    C, h = 64, p["heads"]
    last = x[:, -1:].contiguous()
    qkv = ops.gemm(ops.layernorm(last, p["g1"], p["b1"], 1e-6), p["wqkv"])
    qn, kn = qkv[..., :C], qkv[..., C:2 * C]
    ops.rope3d(qn, kn, pos[-1:], freqs, p["sections"], h, out=(qn, kn))
    K, V = torch.cat([k[:, :-1], kn], 1), torch.cat([v[:, :-1], qkv[..., 2 * C:]], 1)
    y = ops.gemm(ops.attention(qn, K, V, h, (C // h) ** -0.5), p["wo"], residual=last)
    hid = ops.gated_ffn(ops.layernorm(y, p["g2"], p["b2"], 1e-6), p["wgu"], p["bgu"])
    z = ops.gemm(hid, p["wd"], residual=y)
    _within(z, ref[:, -1:], tol, "newest token")


def test_video_block_served_in_8_bits(cuda):
    """The block's projections as 8-bit products.  Each of two factors carries a rounding of half a step of 1/127 of its
    row's largest value (about 3 sigma): relative error of a product about sqrt(2) * 3 / 127 / sqrt(12) = 1 %; four
    products in a chain, so 5 % in the mean square."""
    ops = _ops()
    p, pos = _params(torch.float16), _grid(2, 5, 5)
    x = _rand(3, 50, 64, dt=torch.float16, seed=20)
    freqs = ops.rope3d_freqs(p["sections"])
    w8 = {n: ops.quant_rows(p[n]) for n in ("wqkv", "wo", "wd")}
    lin = lambda t, n, **kw: ops.gemm_i8(*ops.quant_rows(t), *w8[n], **kw)  # noqa: E731
    C, h = 64, p["heads"]
    qkv = lin(ops.layernorm(x, p["g1"], p["b1"], 1e-6), "wqkv")
    q, k = qkv[..., :C], qkv[..., C:2 * C]
    ops.rope3d(q, k, pos, freqs, p["sections"], h, out=(q, k))
    y = lin(ops.attention(q, k, qkv[..., 2 * C:], h, (C // h) ** -0.5), "wo", residual=x)
    z = lin(ops.gated_ffn(ops.layernorm(y, p["g2"], p["b2"], 1e-6), p["wgu"], p["bgu"]), "wd", residual=y)
    ref = _block_ref(x.to(F64), pos, freqs, {n: t.to(F64) if torch.is_tensor(t) else t for n, t in p.items()})
    assert float((z.to(F64) - ref).norm() / ref.norm()) < 0.05


def test_captured_replayed_and_on_other_streams(cuda):
    """All operators captured in two graphs, replayed in turn with new inputs and eager work between, equal the eager
    results every time; and on a side stream."""
    ops = _ops()
    dt = torch.bfloat16
    M, H, K, N = 70, 61, 72, 40
    sec, freqs = (4, 4, 4), ops.rope3d_freqs((4, 4, 4))
    pos = _grid(7, 5, 2)
    w = _rand(2 * H, K, dt=dt, seed=1)
    wq, ws = ops.quant_rows(_rand(N, K, dt=dt, seed=2))

    def step(x):
        h, pre = ops.gated_ffn(x, w, save=True)
        g = ops.gated_ffn_bwd(x, w, pre, h)
        q, _ = ops.rope3d(x[None], None, pos, freqs, sec, 3)
        y = ops.gemm_i8(*ops.quant_rows(x), wq, ws, dtype=dt)
        return (h, pre, *g, q, y)

    x = [_rand(M, K, dt=dt, seed=s) for s in (3, 4)]
    step(x[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x[i]))
        graphs.append(g)
    for turn in range(3):
        for i in range(2):
            x[i].copy_(_rand(M, K, dt=dt, seed=10 + 2 * turn + i))
        for i in (0, 1, 0):
            graphs[i].replay()
        want = [step(t) for t in x]
        torch.cuda.synchronize()
        for i in range(2):
            for a, b in zip(outs[i], want[i]):
                assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x[0])
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, step(x[0])):
        assert torch.equal(a, b)


def test_results_do_not_change_from_run_to_run(cuda):
    ops = _ops()
    x, w = _rand(9000, 120, dt=torch.bfloat16, seed=1), _rand(272, 120, dt=torch.bfloat16, seed=2)
    h, pre = ops.gated_ffn(x, w, save=True)
    first = ops.gated_ffn_bwd(x, w, pre, h)
    for _ in range(3):
        for a, b in zip(first, ops.gated_ffn_bwd(x, w, pre, h)):
            assert torch.equal(a, b)


def test_operands_past_32_bits(cuda):
    """Rows, results and gradients that lie more than 4 GiB behind their first: sparse integers, so all of it is exact."""
    ops = _ops()
    M, K, H, dt = (1 << 20) + 70, 2112, 1056, torch.bfloat16
    at = torch.tensor([0, 77, 1 << 19, (1 << 20) - 1, M - 1], device="cuda")
    x = torch.zeros(M, K, device="cuda", dtype=dt)
    x[at] = _ints(len(at), K, dt=dt, seed=1)
    w = _ints(2 * H, K, dt=dt, seed=2)
    h, pre = ops.gated_ffn(x, w, act="relu", save=True)                 # x, pre 4.4 GB
    assert torch.equal(h[at], ops.gated_ffn(x[at], w, act="relu")) and int(h.any(1).sum()) <= len(at)
    dh = torch.zeros(M, H, device="cuda", dtype=dt)
    dh[at] = _ints(len(at), H, dt=dt, seed=3)
    got, ref = ops.gated_ffn_bwd(x, w, pre, dh, act="relu"), ops.gated_ffn_bwd(x[at], w, pre[at], dh[at], act="relu")
    assert torch.equal(got[0][at], ref[0]) and int(got[0].any(1).sum()) <= len(at)
    assert torch.equal(got[2], ref[2])
    # dW in either order of its few terms: f32 sums of at most five 16-bit products, each partial sum rounded, then once
    tol = pre[at].float().abs().amax() * 5 * 4 * 2.0 ** -24
    _within(got[1], ref[1].to(F64), tol + 2 * U[dt] * ref[1].to(F64).abs(), "dW")
    del got, h, pre, dh
    q = x.view(M, K)[None]
    pos = torch.zeros(M, 3, device="cuda", dtype=torch.int32)
    pos[at] = torch.tensor([3, 5, 7], device="cuda", dtype=torch.int32)
    freqs = ops.rope3d_freqs((4, 4, 4))
    y = ops.rope3d(q, None, pos, freqs, (4, 4, 4), K // 32)[0]
    assert torch.equal(y[0, at], ops.rope3d(q[:, at], None, pos[at], freqs, (4, 4, 4), K // 32)[0][0])
    assert int(y[0].any(1).sum()) <= len(at)
    del y
    a = torch.zeros(2 * M, K, device="cuda", dtype=torch.int8)
    a[2 * at] = _codes(len(at), K, 5)
    b, s = _codes(64, K, 6), torch.ones(2 * M, device="cuda")
    y = ops.gemm_i8(a, s, b, s[:64], dtype=torch.float32)
    assert torch.equal(y[2 * at], ops.gemm_i8(a[2 * at], s[:5], b, s[:64], dtype=torch.float32))
    assert int(y.any(1).sum()) <= len(at)


@pytest.mark.parametrize("M", [3, 70, 300])
def test_weights_of_almost_4_gib(cuda, M):
    """The largest weights that are taken (the offset of the last row is just under 2^32), all of it exact."""
    ops = _ops()
    N, K = (1 << 20) + 4096 + 40, 4064
    assert N * K < 1 << 32 <= (N + 8192) * K
    w = torch.zeros(N, K, device="cuda", dtype=torch.int8)
    at = torch.tensor([0, 5000, 1 << 19, (1 << 20) + 1, N - 2, N - 1], device="cuda")
    w[at] = _codes(len(at), K, 1)
    a, one = _codes(M, K, 2), torch.ones(N, device="cuda")
    y = ops.gemm_i8(a, one[:M], w, one, dtype=torch.float32)
    ref = (a.cpu().double() @ w[at].cpu().double().t()).float().cuda()
    assert torch.equal(y[:, at], ref) and int(y.any(0).sum()) <= len(at)
    del w, y
    H, K = N // 2, 2032
    w = torch.zeros(2 * H, K, device="cuda", dtype=torch.bfloat16)
    at = torch.tensor([0, 5000, 1 << 18, H - 2, H - 1], device="cuda")
    w[at], w[H + at] = (_ints(len(at), K, dt=torch.bfloat16, seed=s) for s in (3, 4))
    x = _ints(M, K, dt=torch.bfloat16, seed=5)
    h = ops.gated_ffn(x, w, act="relu")
    g, u = ((x.cpu().double() @ w[i].cpu().double().t()) for i in (at, H + at))
    # the product of two integers under 2^11 is exact in f32
    assert torch.equal(h[:, at], (g.relu() * u).to(torch.bfloat16).cuda()) and int(h.any(0).sum()) <= len(at)
