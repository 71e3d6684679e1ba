"""GPU: cross attention to states of another length, RMS norm with residual and 8-bit output, gradient norm and clipping (ogmm_amd.ops, train_ops, Trainer)
against plain evaluations in 64 bits.

Tolerances are elementwise and count roundings.  u = 2^-24 is fp32's half step, h(t) the half step of the tensors' type (bf16 2^-8, fp16 2^-11, fp32 u)."""
import math

import pytest
import torch

import ogmm_amd          # (before anything touches the GPU: it switches the runtime's graph packet capture off)

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = {torch.float32: "fp32", torch.bfloat16: "bf16", torch.float16: "fp16"}


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """the absolute half step below the type's normal numbers (matters for fp16 alone)"""
    return 2.0 ** -25 if t == torch.float16 else 0.0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def close(got, want, tol, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= tol)          # (a NaN is bad)
    assert not bad.any(), "%s: %d of %d values beyond the bound; worst %.3g at a bound of %.3g" % (
        what, int(bad.sum()), bad.numel(), float(off[bad].max()), float((tol if torch.is_tensor(tol) else torch.tensor(tol)).expand_as(off)[bad].min()))


# ---------------------------------------------------------------------------------------------- cross attention
def attention_case(B, Nq, Nk, H, G, d, dtype, seed, size=1.5):
    g = gen(seed)
    return randn(g, B, Nq, H, d, dtype=torch.float32).mul(size).to(dtype), randn(g, B, Nk, H // G, d, dtype=dtype), randn(g, B, Nk, H // G, d, dtype=dtype), randn(g, B, Nq, H, d, dtype=dtype)


def reference(q, k, v, do, kv_lens=None, q_lens=None, key_mask=None, scale=None, grads=True, stored=True):
    """values and elementwise bounds in 64 bits: {name: (value, bound)}; stored = False: o is known to h^2 (its rounding and the rounding of what that left)"""
    B, Nq, H, d = q.shape
    Nk, Hkv = k.shape[1:3]
    G, t = H // Hkv, q.dtype
    scale = d ** -0.5 if scale is None else scale
    ok = torch.ones(B, Nk, dtype=torch.bool, device="cuda")
    if kv_lens is not None:
        ok &= torch.arange(Nk, device="cuda")[None] < kv_lens.clamp(0, Nk)[:, None]
    if key_mask is not None:
        ok &= key_mask
    rows = torch.ones(B, Nq, dtype=torch.bool, device="cuda") if q_lens is None else torch.arange(Nq, device="cuda")[None] < q_lens.clamp(0, Nq)[:, None]
    zero_k, zero_q = ~ok[:, :, None, None], ~rows[:, :, None, None]

    def heads(x):
        return x.permute(0, 2, 1, 3).contiguous()          # [B, heads, n, d]

    Q = heads(q.double().masked_fill(zero_q, 0.0))
    DO = heads(do.double().masked_fill(zero_q, 0.0)) if grads else None
    K, V = (heads(x.double().masked_fill(zero_k, 0.0)).repeat_interleave(G, dim=1) for x in (k, v))
    see = ok[:, None, None, :] & rows[:, None, :, None]
    S = (Q @ K.transpose(2, 3).contiguous() * scale).masked_fill(~see, -math.inf)
    m = S.amax(dim=3, keepdim=True)
    any_key = m > -math.inf
    m = m.masked_fill(~any_key, 0.0)
    P = torch.exp(S - m)
    L = P.sum(dim=3, keepdim=True)
    lse = torch.where(any_key, m + torch.log(L), torch.full_like(m, -math.inf))[..., 0]
    P = P / L.masked_fill(L == 0, 1.0)
    O = P @ V
    h, a = half_step(t), tiny(t)
    # a score: d products and sums and the scaling in fp32, the exponential's argument and its own steps (2 u each), at the size of the products' magnitudes
    ds = (d + 8) * U * (Q.abs() @ K.abs().transpose(2, 3).contiguous() * abs(scale)).amax(dim=3, keepdim=True) + 8 * U
    rel_p = 2 * ds + (Nk + 16) * U          # numerator and denominator, the sum over the keys and the rescalings of the running one
    half_p = h if t != torch.float32 else 0.0          # P as an operand of the type's matrix instruction
    e_o = (rel_p + half_p + Nk * U) * (P @ V.abs()) + a * V.abs().sum(dim=2, keepdim=True) + (h if stored else h * h) * O.abs() + a

    def back(x):
        return x.permute(0, 2, 1, 3)

    out = {"o": (back(O), back(e_o)), "lse": (lse, torch.where(any_key[..., 0], ds[..., 0] + (Nk + 16) * U + 4 * U * lse.abs(), torch.zeros_like(lse)))}
    if not grads:
        return out
    dP = DO @ V.transpose(2, 3).contiguous()
    D = (DO * O).sum(dim=3, keepdim=True)
    dS = P * (dP - D)
    # D from the stored o (bound e_o), dP: d products and sums
    e_d = (DO.abs() * (e_o + (d + 4) * U * O.abs())).sum(dim=3, keepdim=True)
    e_dp = (d + 4) * U * (DO.abs() @ V.abs().transpose(2, 3).contiguous())
    # the backward forms P from the stored log sum exp: its error on top of the score's
    rel_pb = ds + out["lse"][1][..., None] + 8 * U
    e_ds = P * (e_d + e_dp + U * (dP.abs() + D.abs())) + (rel_pb + half_p) * dS.abs()
    # fp16: dS is held as a power of two times itself that follows max|dO| over the rows that share a key head: the half step of its smallest values moves with it
    top = DO.abs().amax(dim=(2, 3), keepdim=True).view(B, Hkv, G, 1, 1).amax(dim=2, keepdim=True).expand(B, Hkv, G, 1, 1).reshape(B, H, 1, 1)
    e_ds = e_ds + 2 * a * top * (P > 0)
    dQ = dS @ K * scale
    e_dq = abs(scale) * (e_ds @ K.abs() + (Nk + 8) * U * (dS.abs() @ K.abs())) + h * dQ.abs() + a

    def shared(x):          # sum over the query heads of a key head
        return x.view(B, Hkv, G, Nk, d).sum(dim=2)

    T = lambda x: x.transpose(2, 3).contiguous()  # noqa: E731
    dK, dV = shared(T(dS) @ Q) * scale, shared(T(P) @ DO)
    sums = (Nq * G + 8) * U
    e_dk = abs(scale) * shared(T(e_ds) @ Q.abs() + sums * (T(dS).abs() @ Q.abs())) + h * dK.abs() + a
    e_dv = shared(T(P * (rel_pb + half_p)) @ DO.abs() + sums * (T(P) @ DO.abs())) + a * shared(DO.abs().sum(dim=2, keepdim=True).expand(B, H, Nk, d)) + h * dV.abs() + a
    out.update(dq=(back(dQ), back(e_dq)), dk=(back(dK), back(e_dk)), dv=(back(dV), back(e_dv)))
    return out


def check_attention(q, k, v, do, grads=True, **kw):
    from ogmm_amd import ops
    want = reference(q, k, v, do, grads=grads, **kw)
    o, lse = ops.cross_attention(q, k, v, need_lse=True, **kw)
    assert torch.equal(ops.cross_attention(q, k, v, **kw), o)
    close(o, *want["o"], "o")
    empty = want["lse"][0] == -math.inf
    assert bool((lse[empty] == -math.inf).all())
    close(lse[~empty], want["lse"][0][~empty], want["lse"][1][~empty], "lse")
    if grads:
        got = ops.cross_attention_bwd(q, k, v, o, lse, do, **kw)
        for name, x in zip(("dq", "dk", "dv"), got):
            close(x, *want[name], name)
        for x, y in zip(got, ops.cross_attention_bwd(q, k, v, o, lse, do, **kw)):
            assert torch.equal(x, y), "a repeated call differs"
        # with what the rounding of o left: D is as in fp32
        o2, lse2, rest = ops.cross_attention(q, k, v, need_lse=True, need_rest=True, **kw)
        assert torch.equal(o2, o) and torch.equal(lse2, lse) and (rest is None) == (q.dtype == torch.float32)
        if rest is not None:
            close(o.double() + rest.double(), *reference(q, k, v, do, grads=False, stored=False, **kw)["o"], "o + rest")
        want = reference(q, k, v, do, stored=False, **kw)
        for name, x in zip(("dq", "dk", "dv"), ops.cross_attention_bwd(q, k, v, o, lse, do, rest=rest, **kw)):
            close(x, *want[name], name + " with the rest")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("B,Nq,Nk,H,G,d", [
    (1, 1, 1, 1, 1, 8), (2, 1, 717, 4, 1, 128), (1, 3, 65, 8, 8, 64), (2, 33, 31, 2, 2, 40), (1, 128, 128, 4, 1, 128), (2, 129, 257, 4, 2, 96),
    (1, 64, 1, 2, 1, 32), (3, 200, 333, 6, 3, 72), (1, 5, 2048, 16, 4, 128), (1, 257, 100, 1, 1, 16), (1, 1, 5000, 2, 2, 64), (1, 70, 640, 5, 5, 120)])
def test_attention_sizes(dtype, B, Nq, Nk, H, G, d):
    check_attention(*attention_case(B, Nq, Nk, H, G, d, dtype, 7 * Nq + Nk))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("Nq,G", [(1, 4), (70, 2), (260, 1)])
def test_attention_lengths_and_masks(dtype, Nq, G):
    """ragged keys and rows, lengths of zero and one and beyond the padded ones, a mask that leaves a batch entry nothing; NaN and infinities wherever nothing may look"""
    B, Nk, H, d = 6, 300, 4, 64
    q, k, v, do = attention_case(B, Nq, Nk, H, G, d, dtype, 11)
    kv_lens = torch.tensor([0, 1, 300, 129, 1000, 64], dtype=torch.int32, device="cuda")
    q_lens = torch.tensor([Nq, 1, Nq // 2, Nq + 5, Nq, -3], dtype=torch.int32, device="cuda")
    mask = torch.rand(B, Nk, generator=gen(5), device="cuda") < 0.7
    mask[3] = False
    mask[4, 128:256] = False          # whole tiles of keys without one
    for kw in (dict(kv_lens=kv_lens), dict(key_mask=mask), dict(kv_lens=kv_lens, q_lens=q_lens, key_mask=mask)):
        ok = torch.ones(B, Nk, dtype=torch.bool, device="cuda")
        if "kv_lens" in kw:
            ok &= torch.arange(Nk, device="cuda")[None] < kv_lens[:, None]
        ok &= kw.get("key_mask", ok)
        k2, v2 = k.clone(), v.clone()
        k2[~ok] = math.nan
        v2[~ok] = math.inf
        q2, do2 = q.clone(), do.clone()
        if "q_lens" in kw:
            behind = torch.arange(Nq, device="cuda")[None] >= q_lens[:, None]
            q2[behind] = math.inf
            do2[behind] = math.nan
        check_attention(q2, k2, v2, do2, **kw)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_attention_scores_far_apart(dtype):
    """scores of hundreds: every row is nearly one key, running maxima move by much; and a negative scale"""
    q, k, v, do = attention_case(1, 100, 400, 2, 1, 64, dtype, 3, size=24.0)
    check_attention(q, k, v, do)
    check_attention(q, k, v, do, scale=-0.05)
    check_attention(q, k, v, do, scale=0.0)


def test_attention_small_gradients_in_fp16():
    """an upstream gradient far below fp16's normal products"""
    q, k, v, do = attention_case(1, 130, 300, 4, 2, 64, torch.float16, 9)
    check_attention(q, k, v, (do.float() * 2.0 ** -10).half())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_attention_strides(dtype):
    """heads first in memory, a slice of a wider projection, one sequence expanded over the batch, an address and a step that are not multiples of 16 bytes"""
    B, Nq, Nk, H, d = 2, 40, 90, 4, 64
    g = gen(21)
    q = randn(g, B, H, Nq, d, dtype=dtype).transpose(1, 2)
    kv = randn(g, B, Nk, 2, H, d, dtype=dtype)
    do = randn(g, B, Nq, H, d, dtype=dtype)
    check_attention(q, kv[:, :, 0], kv[:, :, 1], do)
    one = randn(g, 1, Nk, H, d, dtype=dtype).expand(B, Nk, H, d)
    check_attention(q, one, one, do.transpose(1, 2).contiguous().transpose(1, 2))
    odd = randn(g, B * Nk * (H * d + 1) + 1, dtype=dtype)[1:].as_strided((B, Nk, H, d), (Nk * (H * d + 1), H * d + 1, d, 1))
    check_attention(q, odd, odd, do)
    mask = (torch.rand(Nk, B, generator=g, device="cuda") < 0.5).t()
    check_attention(q, one, odd, do, key_mask=mask)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_attention_autograd_matches_differences(dtype):
    from ogmm_amd import train_ops
    q, k, v, do = attention_case(1, 9, 20, 2, 2, 16, dtype, 4)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    mask = torch.ones(1, 20, dtype=torch.bool, device="cuda")
    mask[0, 3] = False
    o = train_ops.cross_attention(*leaves, key_mask=mask)
    grads = torch.autograd.grad(o, leaves, do)
    g = gen(6)

    def value(ts):
        return float((reference(*ts, do, key_mask=mask, grads=False)["o"][0] * do.double()).sum())

    for i in range(3):
        way = randn(g, *leaves[i].shape).double()
        ts = [t.detach().double() for t in leaves]
        e = 1e-5
        up = value([t + e * way if j == i else t for j, t in enumerate(ts)])
        down = value([t - e * way if j == i else t for j, t in enumerate(ts)])
        along = (grads[i].double() * way).sum()
        bound = (reference(q, k, v, do, key_mask=mask)[("dq", "dk", "dv")[i]][1] * way.abs()).sum()
        assert abs(float(along) - (up - down) / (2 * e)) <= float(bound) + 1e-6 * float(grads[i].double().norm() * way.norm())


def test_attention_nothing():
    from ogmm_amd import ops
    for B, Nq, Nk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k, v, do = attention_case(B, Nq, Nk, 2, 1, 32, torch.bfloat16, 1)
        o, lse = ops.cross_attention(q, k, v, need_lse=True)
        dq, dk, dv = ops.cross_attention_bwd(q, k, v, o, lse, do)
        for t in (o, dq, dk, dv):
            assert not t.numel() or float(t.abs().max()) == 0.0
        assert bool((lse == -math.inf).all())


def test_attention_gradient_with_more_scores_than_are_kept():
    """fp32 keeps dS between its two kernels up to 2^28 scores; these are more, and the second kernel forms them again"""
    q, k, v, do = attention_case(1, 8200, 16400, 2, 2, 8, torch.float32, 11)
    mask = torch.rand(1, 16400, generator=gen(12), device="cuda") < 0.7
    lens = torch.tensor([16333], dtype=torch.int32, device="cuda"), torch.tensor([8190], dtype=torch.int32, device="cuda")
    check_attention(q, k, v, do, kv_lens=lens[0], q_lens=lens[1], key_mask=mask)


def test_attention_offsets_past_31_bits():
    """a cache of more than 2^31 bytes' and 2^31 elements' worth of keys: the last batch entry's rows are read where they are"""
    B, Nk, Hkv, d = 17, 16384 * 8, 8, 128          # 17 x 134 217 728 elements, 4.6 GB each for k and v
    k = torch.zeros(B, Nk, Hkv, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    g = gen(2)
    n = 700
    for t in (k, v):
        t[-1, -n:] = randn(g, n, Hkv, d, dtype=torch.bfloat16)
    mask = torch.zeros(B, Nk, dtype=torch.bool, device="cuda")
    mask[:, -n:] = True
    q = randn(g, B, 1, 2 * Hkv, d, dtype=torch.bfloat16)
    from ogmm_amd import ops
    o = ops.cross_attention(q, k, v, key_mask=mask)
    want = reference(q[-1:], k[-1:, -n:], v[-1:, -n:], q[-1:], grads=False)["o"]
    close(o[-1:], *want, "o")
    assert float(o[:-1].abs().max()) == 0.0


# ---------------------------------------------------------------------------------------------- RMS norm
def norm_reference(x, w, r, eps):
    h = x.double() + (0 if r is None else r.double())
    rstd = 1 / ((h * h).mean(dim=-1, keepdim=True) + eps).sqrt()
    return h, rstd, h * rstd * w.double()


# a row's sum of squares: at most 32 values in a lane, six exchanges, sixteen waves; half of that in rstd; the residual's sum, the products
NORM_U = 40 * U


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("D", [1, 3, 16, 63, 64, 129, 512, 717, 1024, 1500, 2049, 4096, 5003, 8192, 12289, 32768])
def test_norm_widths(dtype, D):
    from ogmm_amd import ops
    for R, residual, wtype in ((1, True, dtype), (7, False, torch.float32), (33, True, torch.float32)):
        g = gen(D + R)
        x, r = randn(g, R, D, dtype=dtype), randn(g, R, D, dtype=dtype) if residual else None
        w = (1 + 0.3 * randn(g, D)).to(wtype)
        y, h, rstd = ops.rms_norm(x, w, r, eps=1e-5)
        H, RS, Y = norm_reference(x, w, r, 1e-5)
        close(y, Y, (NORM_U + half_step(dtype)) * Y.abs() + tiny(dtype), "y")
        close(rstd, RS[:, 0], NORM_U * RS[:, 0], "rstd")
        if residual:
            close(h, H, half_step(dtype) * H.abs() + tiny(dtype), "h")
        else:
            assert h is x


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("R,D", [(1, 5), (3, 64), (2000, 100), (37, 512), (700, 717), (1500, 1030), (90, 4097), (40, 16384), (9, 32768)])
def test_norm_gradient(dtype, R, D):
    from ogmm_amd import ops
    g = gen(R * D)
    h, dy, dh = (randn(g, R, D, dtype=dtype) for _ in range(3))
    w = (1 + 0.3 * randn(g, D)).to(dtype)
    _, rs, _ = norm_reference(h, w, None, 1e-6)
    rstd = rs[:, 0].float()
    for with_dh in (False, True):
        dx, dw = ops.rms_norm_bwd(dy, h, w, rstd, dh if with_dh else None)
        G, XH = dy.double() * w.double(), h.double() * rs
        mean = (G * XH).mean(dim=1, keepdim=True)
        DX = rs * (G - XH * mean) + (dh.double() if with_dh else 0)
        size = rs * (G.abs() + XH.abs() * (G * XH).abs().mean(dim=1, keepdim=True)) + (dh.double().abs() if with_dh else 0)
        close(dx, DX, 72 * U * size + half_step(dtype) * DX.abs() + tiny(dtype), "dx")
        DW = (dy.double() * XH).sum(dim=0)
        close(dw, DW, (min(R, 64 + R // 64) + 48) * U * (dy.double() * XH).abs().sum(dim=0) + half_step(dtype) * DW.abs() + tiny(dtype), "dw")
        again = ops.rms_norm_bwd(dy, h, w, rstd, dh if with_dh else None)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS.get)
@pytest.mark.parametrize("R,D", [(1, 3), (102, 458), (50, 130), (33, 1024), (20, 5003), (12, 16384), (9, 32768)])
def test_norm_gradient_from_the_summands(dtype, R, D):
    """x and residual in place of their stored sum: the gradients are those of the sum itself, and so through autograd"""
    from ogmm_amd import ops, train_ops
    g = gen(R + D)
    x, r, dy, dh = (randn(g, R, D, dtype=dtype) for _ in range(4))
    w = (1 + 0.3 * randn(g, D)).to(dtype)
    _, h, rstd = ops.rms_norm(x, w, r)
    H, RS, _ = norm_reference(x, w, r, 1e-6)
    G, XH = dy.double() * w.double(), H * RS
    DX = RS * (G - XH * (G * XH).mean(dim=1, keepdim=True)) + dh.double()
    size = RS * (G.abs() + XH.abs() * (G * XH).abs().mean(dim=1, keepdim=True)) + dh.double().abs()
    DW = (dy.double() * XH).sum(dim=0)
    dx, dw = ops.rms_norm_bwd(dy, x, w, rstd, dh, residual=r)
    # as test_norm_gradient, with rstd known to NORM_U and the sum to U: 41 U for each of the three factors of xh mean(g xh)
    close(dx, DX, (72 + 3 * 41) * U * size + half_step(dtype) * DX.abs() + tiny(dtype), "dx")
    close(dw, DW, (min(R, 64 + R // 64) + 48 + 41) * U * (dy.double() * XH).abs().sum(dim=0) + half_step(dtype) * DW.abs() + tiny(dtype), "dw")
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    grads = torch.autograd.grad(train_ops.rms_norm(leaves[0], leaves[2], leaves[1]), leaves, (dy, dh))
    assert torch.equal(grads[0], dx) and torch.equal(grads[1], dx) and torch.equal(grads[2], dw)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_norm_autograd_matches_differences(dtype):
    from ogmm_amd import train_ops
    g = gen(8)
    x, r, w = randn(g, 4, 5, 24, dtype=dtype), randn(g, 4, 5, 24, dtype=dtype), (1 + 0.3 * randn(g, 24)).to(dtype)
    dy, dh = randn(g, 4, 5, 24, dtype=dtype), randn(g, 4, 5, 24, dtype=dtype)
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y, h = train_ops.rms_norm(leaves[0], leaves[2], leaves[1])
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))
    assert torch.equal(grads[0], grads[1])

    def value(ts):
        H, _, Y = norm_reference(ts[0].view(20, 24), ts[2], ts[1].view(20, 24), 1e-6)
        return float((Y * dy.double().view(20, 24)).sum() + (H * dh.double().view(20, 24)).sum())

    for i in range(3):
        way = randn(g, *leaves[i].shape).double()
        ts = [t.detach().double() for t in leaves]
        e = 1e-5
        ends = [value([t + s * e * way if j == i else t for j, t in enumerate(ts)]) for s in (1, -1)]
        along = float((grads[i].double() * way).sum())
        # the stored sum and each gradient are rounded once: values of order |dy| + |dh| <= 8, each of the three terms by h at most
        bound = 24 * (half_step(dtype) + 64 * U) * float(way.abs().sum()) * (1 if i < 2 else 20)
        assert abs(along - (ends[0] - ends[1]) / (2 * e)) <= bound + 1e-5
    # one of the two outputs alone, and no residual
    only_y = torch.autograd.grad(train_ops.rms_norm(leaves[0], leaves[2], leaves[1])[0], leaves, dy)
    H, RS, _ = norm_reference(x, w, r, 1e-6)
    assert float((only_y[0].double() - (grads[0].double() - dh.double())).abs().max()) <= 8 * half_step(dtype) * 8
    only_h = torch.autograd.grad(train_ops.rms_norm(leaves[0], leaves[2], leaves[1])[1], leaves[:2], dh)
    assert torch.equal(only_h[0], dh) and torch.equal(only_h[1], dh)
    plain = train_ops.rms_norm(leaves[0], leaves[2])
    assert plain.shape == x.shape and len(torch.autograd.grad(plain, (leaves[0], leaves[2]), dy)) == 2


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("group", [0, 32, 64, 128])
@pytest.mark.parametrize("R,D", [(1, 1), (5, 50), (40, 512), (21, 717), (3, 2500), (2, 9000), (2, 32768)])
def test_norm_eight_bits(dtype, group, R, D):
    from ogmm_amd import ops
    g = gen(R + D + group)
    x, r = randn(g, R, D, dtype=dtype), randn(g, R, D, dtype=dtype)
    w = (1 + 0.3 * randn(g, D)).to(dtype)
    if R > 2:
        x[1] = 0
        r[1] = 0          # a row of zeros
        x[2] *= 100.0
    q, s, h = ops.rms_norm_q8(x, w, r, eps=1e-6, group=group)
    H, _, Y = norm_reference(x, w, r, 1e-6)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32
    close(h, H, half_step(dtype) * H.abs() + tiny(dtype), "h")
    width = group or D
    S = torch.stack([Y[:, i:i + width].abs().amax(dim=1) for i in range(0, D, width)], dim=1) / 448.0
    close(s, S, (NORM_U + 4 * U) * S, "scales")
    each = s.double().repeat_interleave(width, dim=1)[:, :D]
    # to nearest: half a step of four bits relative, or half of the smallest step 2^-9 of the scaled values
    close(q.double() * each, Y, torch.maximum(2.0 ** -4 * Y.abs(), 2.0 ** -10 * each) * (1 + 2.0 ** -8) + 2 * NORM_U * Y.abs(), "q scales")
    top = (q.double().abs()).amax(dim=1)
    assert bool(((top == 448.0) | (S[:, 0] == 0) | (group > 0)).all())
    q2, s2, x2 = ops.rms_norm_q8(x, w, eps=1e-6, group=group)
    assert x2 is x and q2.shape == q.shape and s2.shape == s.shape


def test_norm_values_at_the_ends():
    """magnitudes whose squares or scales leave the small numbers, zeros, a NaN row beside others"""
    from ogmm_amd import ops
    x = torch.full((4, 96), 1e-30, device="cuda")
    x[1] = 0.0
    x[2, 5] = math.nan
    x[3] = 1e18
    w = torch.ones(96, device="cuda")
    y, _, _ = ops.rms_norm(x, w, eps=0.0)
    assert bool(torch.isnan(y[2]).all()) and float((y[3] - 1).abs().max()) < 1e-5
    y, _, _ = ops.rms_norm(x, w, eps=1e-6)
    assert float((y[0] - 1e-27).abs().max()) < 1e-31 and float(y[1].abs().max()) == 0.0
    q, s, _ = ops.rms_norm_q8(x, w, eps=1e-6)
    assert float(q[1].float().abs().max()) == 0.0 and float(s[1]) == 0.0 and bool(torch.isnan(s[2]).all())
    assert float((q[0].float() * s[0] - 1e-27).abs().max()) < 1e-30
    q, s, _ = ops.rms_norm_q8(x[:1], w * 1e-13, eps=1e-6)          # y = 1e-40: below the normal numbers
    assert float(q.float().abs().max()) == 0.0 and float(s.abs().max()) == 0.0


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_norm_strides_and_shapes(dtype):
    from ogmm_amd import ops
    g = gen(31)
    wide = randn(g, 50, 301, dtype=dtype)
    w = (1 + 0.3 * randn(g, 200)).to(dtype)
    x, r = wide[:, 1:201], wide[:, 101:301]
    y, h, rstd = ops.rms_norm(x, w, r)
    y2, h2, rstd2 = ops.rms_norm(x.contiguous(), w, r.contiguous())
    assert torch.equal(y, y2) and torch.equal(h, h2) and torch.equal(rstd, rstd2)
    dx, dw = ops.rms_norm_bwd(r, x, w, rstd, x)
    dx2, dw2 = ops.rms_norm_bwd(r.contiguous(), x.contiguous(), w, rstd, x.contiguous())
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)
    t = randn(g, 200, 50, dtype=dtype).t()
    assert torch.equal(ops.rms_norm(t, w)[0], ops.rms_norm(t.contiguous(), w)[0])
    row = randn(g, 1, 200, dtype=dtype).expand(6, 200)
    assert torch.equal(ops.rms_norm(row, w)[0], ops.rms_norm(row.contiguous(), w)[0])
    one = ops.rms_norm(wide[0, :200], w)
    assert one[0].shape == (200,) and one[2].shape == () and torch.equal(one[0], ops.rms_norm(wide[:1, :200], w)[0][0])
    none = ops.rms_norm(wide[:0, :200], w, wide[:0, :200])
    assert none[0].shape == (0, 200)
    dx, dw = ops.rms_norm_bwd(wide[:0, :200], wide[:0, :200], w, none[2])
    assert dx.shape == (0, 200) and float(dw.abs().max()) == 0.0
    assert ops.rms_norm_q8(wide[:0, :200], w, group=64)[1].shape == (0, 4)


# ---------------------------------------------------------------------------------------------- gradient norm and clipping
def grad_tensors(g, sizes, types):
    return [randn(g, n).mul(10.0 ** -(i % 5)).to(types[i % len(types)]) for i, n in enumerate(sizes)]


SIZES = [1, 2, 7, 8, 4095, 4096, 4097, 100_003, 0, 31, 65_536, 1_000_003]


@pytest.mark.parametrize("types", [[torch.float32], [torch.bfloat16], [torch.float16], TYPES], ids=["fp32", "bf16", "fp16", "mixed"])
@pytest.mark.parametrize("many", [1, 20])          # (20: more tensors than the kernel arguments hold at once)
def test_gradients(types, many):
    from ogmm_amd import ops
    g = gen(13)
    grads = grad_tensors(g, SIZES * many, types)
    total = math.sqrt(sum(float(x.double().square().sum()) for x in grads))
    assert abs(float(ops.grad_norm(grads)) - total) <= 2 * U * total
    assert abs(float(ops.grad_norm(grads, inv_scale=0.125)) - total / 8) <= 2 * U * total / 8
    before = [x.clone() for x in grads]
    # under the limit: nothing moves
    assert abs(float(ops.clip_grads_(grads, 2 * total)) - total) <= 2 * U * total
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    # out of place, un-scaled and clipped
    out = [torch.full(x.shape, math.nan, device="cuda") for x in grads]
    norm = ops.clip_grads_(grads, 0.01, inv_scale=2.0 ** -4, out=out)
    f = 0.01 / (total / 16 + 1e-6) / 16
    assert abs(float(norm) - total / 16) <= 2 * U * total / 16
    for a, b, o in zip(grads, before, out):
        assert torch.equal(a, b)
        close(o, b.double() * f, 4 * U * b.double().abs() * f, "out")
    # in place
    ops.clip_grads_(grads, 0.01, inv_scale=2.0 ** -4)
    for a, b in zip(grads, before):
        close(a, b.double() * f, (4 * U + half_step(a.dtype)) * b.double().abs() * f + tiny(a.dtype), "in place")
    # un-scaling alone
    grads = [x.clone() for x in before]
    ops.clip_grads_(grads, math.inf, inv_scale=0.5)
    assert all(torch.equal(a, (b.float() * 0.5).to(b.dtype)) for a, b in zip(grads, before))


def test_gradients_at_odd_addresses():
    from ogmm_amd import ops
    g = gen(17)
    for t in TYPES:
        bucket = randn(g, 50_000, dtype=t)
        grads = [bucket[1:4], bucket[5:20_006], bucket[20_007:49_999]]
        copy = [x.clone() for x in grads]
        guard = [int(i) for i in (0, 4, 20_006, 49_999)]
        kept = bucket[guard].clone()
        total = math.sqrt(sum(float(x.double().square().sum()) for x in grads))
        f = 1.0 / (total + 1e-6)
        flat = torch.full((50_001,), math.nan, device="cuda")
        out = [flat[3:6], flat[7:20_008], flat[20_009:50_001]]
        ops.clip_grads_(grads, 1.0, out=out)
        ops.clip_grads_(grads, 1.0)
        for a, b, o in zip(grads, copy, out):
            close(o, b.double() * f, 4 * U * b.double().abs() * f, "out")
            close(a, b.double() * f, (4 * U + half_step(t)) * b.double().abs() * f + tiny(t), "in place")
        assert torch.equal(bucket[guard], kept) and bool(torch.isnan(flat[[0, 1, 2, 6, 20_008]]).all())


def test_gradients_values_at_the_ends():
    from ogmm_amd import ops
    small, large = torch.full((1000,), 1e-30, device="cuda"), torch.full((1000,), 1e30, device="cuda")
    assert abs(float(ops.grad_norm([small])) / (1e-30 * math.sqrt(1000)) - 1) < 4 * U
    assert abs(float(ops.grad_norm([large])) / (1e30 * math.sqrt(1000)) - 1) < 4 * U
    ops.clip_grads_([large], 1.0)
    assert abs(float(large[0]) * math.sqrt(1000) - 1) < 1e-6
    bad = [torch.ones(10, device="cuda"), torch.ones(5000, device="cuda")]
    bad[1][77] = math.nan
    assert math.isnan(float(ops.clip_grads_(bad, 1.0))) and all(bool(torch.isnan(b).all()) for b in bad)
    wide = [torch.ones(10, device="cuda"), torch.ones(5000, device="cuda")]
    wide[1][77] = math.inf
    assert math.isinf(float(ops.clip_grads_(wide, 1.0)))
    assert float(wide[0].abs().max()) == 0.0 and math.isnan(float(wide[1][77])) and float(wide[1][78]) == 0.0
    zero = [torch.zeros(10, device="cuda"), torch.empty(0, device="cuda")]
    assert float(ops.clip_grads_(zero, 1.0)) == 0.0 and float(zero[0].abs().max()) == 0.0
    assert float(ops.clip_grads_([torch.empty(0, device="cuda")], 1.0)) == 0.0
    gone = [torch.ones(3, device="cuda")]
    ops.clip_grads_(gone, 0.0)
    assert float(gone[0].abs().max()) == 0.0
    turned = torch.randn(30, 40, device="cuda").t()
    want = turned.clone() / (float(turned.norm()) + 1e-6)
    ops.clip_grads_(turned, 1.0)
    assert float((turned - want).abs().max()) < 1e-6


# ---------------------------------------------------------------------------------------------- used together, streams, graphs
def block(ops_like, x, r, states, w1, w2, H, **kw):
    """a pre-norm block: residual's sum and norm, attention to the other sequence's states, residual's sum and norm"""
    B, N, D = x.shape
    y, h = ops_like.rms_norm(x, w1, residual=r)
    k, v = states
    o = ops_like.cross_attention(y.view(B, N, H, D // H), k, v, **kw)
    return ops_like.rms_norm(o.reshape(B, N, D), w2, residual=h)


class Plain64:
    @staticmethod
    def rms_norm(x, w, residual, eps=1e-6):
        h = x + residual
        return h / ((h * h).mean(dim=-1, keepdim=True) + eps).sqrt() * w, h

    @staticmethod
    def cross_attention(q, k, v, kv_lens=None):
        G = q.shape[2] // k.shape[2]
        q, k, v = q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(G, 1), v.transpose(1, 2).repeat_interleave(G, 1)
        s = q @ k.transpose(2, 3) * q.shape[3] ** -0.5
        ok = torch.arange(k.shape[2], device=k.device)[None] < kv_lens[:, None]
        return (torch.softmax(s.masked_fill(~ok[:, None, None], -math.inf), dim=3) @ v).transpose(1, 2)


def together(seed, dtype=torch.float32, N=75, Nk=190):
    g = gen(seed)
    B, D, H, Hkv = 3, 256, 4, 2
    x, r = randn(g, B, N, D, dtype=dtype), randn(g, B, N, D, dtype=dtype)
    k, v = randn(g, B, Nk, Hkv, D // H, dtype=dtype), randn(g, B, Nk, Hkv, D // H, dtype=dtype)
    w1, w2 = ((1 + 0.2 * randn(g, D)).to(dtype) for _ in range(2))
    lens = torch.tensor([Nk, 1, Nk // 2], dtype=torch.int32, device="cuda")
    return [x, r, k, v, w1, w2], lens, H, (randn(g, B, N, D, dtype=dtype), randn(g, B, N, D, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_a_block_its_gradient_and_the_clipped_update(dtype):
    from ogmm_amd import ops, train_ops
    tensors, lens, H, up = together(41, dtype)

    def grads_of(kind, ts):
        leaves = [t.clone().requires_grad_() for t in ts]
        x, r, k, v, w1, w2 = leaves
        y, h = block(kind, x, r, (k, v), w1, w2, H, kv_lens=lens)
        return (y.detach(), h.detach()), torch.autograd.grad((y, h), leaves, [u.to(y.dtype) for u in up])

    (y, h), grads = grads_of(train_ops, tensors)
    (Y, Hs), want = grads_of(Plain64, [t.double() for t in tensors])
    # three maps are stored in the type between the operators, and each gradient passes them again: a relative error of 8 half steps in the 2-norm
    # (fp32: the longest sum, 256 + 190 terms, at u each, twice)
    rel = 8 * half_step(dtype) if dtype != torch.float32 else 2 * (256 + 190) * U
    for a, b in [(y, Y), (h, Hs)] + list(zip(grads, want)):
        assert float((a.double() - b).norm()) <= rel * float(b.norm())
    total = math.sqrt(sum(float(b.square().sum()) for b in want))
    grads = [t.clone() for t in grads]          # (the two summands' gradients are one tensor, which clipping in place would refuse)
    norm = ops.clip_grads_(grads, 0.5)
    assert abs(float(norm) - total) <= rel * total
    assert abs(math.sqrt(sum(float(t.double().square().sum()) for t in grads)) - 0.5) <= (half_step(dtype) + 8 * U) * 0.5 + 1e-6


def test_the_block_serves_single_tokens():
    """one row at a time against the same states gives what the whole sequence gave, within the roundings of both; its rows in 8 bits"""
    from ogmm_amd import ops
    for dtype in TYPES:
        (x, r, k, v, w1, w2), lens, H, _ = together(42, dtype, N=5, Nk=900)
        B, N, D = x.shape

        def serve(x, r):
            y, h, _ = ops.rms_norm(x, w1, r)
            o = ops.cross_attention(y.view(B, -1, H, D // H), k, v, kv_lens=lens)
            return o, h, ops.rms_norm_q8(o.reshape(B, -1, D), w2, h, group=128)

        o, h, (q, s, _) = serve(x, r)
        for n in range(N):
            o1, h1, (q1, s1, _) = serve(x[:, n:n + 1], r[:, n:n + 1])
            assert torch.equal(h1, h[:, n:n + 1])
            assert float((o1.double() - o[:, n:n + 1].double()).norm()) <= 4 * (half_step(dtype) + 64 * U) * float(o[:, n:n + 1].double().norm())
            a, b = (qq.double() * ss.double().repeat_interleave(128, dim=-1) for qq, ss in ((q1, s1), (q[:, n:n + 1], s[:, n:n + 1])))
            assert float((a - b).norm()) <= 2.0 ** -4 * float(b.norm())


def test_side_streams_give_what_the_current_one_gives():
    """two calls of each operator at once, on two streams, and again on the default stream"""
    from ogmm_amd import ops, train_ops
    cases = [together(s, torch.bfloat16) for s in (51, 52)]

    def go(tensors, lens, H, up):
        leaves = [t.clone().requires_grad_() for t in tensors]
        y, h = block(train_ops, leaves[0], leaves[1], leaves[2:4], leaves[4], leaves[5], H, kv_lens=lens)
        grads = [t.clone() for t in torch.autograd.grad((y, h), leaves, up)]
        return [y.detach(), h.detach(), ops.clip_grads_(grads, 0.5)] + grads

    want = [go(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for s, c in zip(streams, cases):
        with torch.cuda.stream(s):
            got.append(go(*c))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_replayed_graph_follows_its_inputs():
    """forward, backward and clipping in one captured graph, replayed on new inputs with eager work between: every replay against the eager result; two graphs side by side"""
    from ogmm_amd import ops
    if not ogmm_amd.graph_replay_safe():
        pytest.skip("the HIP runtime was initialised before graph packet capture could be switched off")

    def go(t, lens, H, up):
        x, r, k, v, w1, w2 = t
        B, N, D = x.shape
        y, h, rstd = ops.rms_norm(x, w1, r)
        q = y.view(B, N, H, D // H)
        o, lse = ops.cross_attention(q, k, v, kv_lens=lens, need_lse=True)
        dq, dk, dv = ops.cross_attention_bwd(q, k, v, o, lse, up[0].view(o.shape), kv_lens=lens)
        dx, dw = ops.rms_norm_bwd(dq.reshape(B, N, D), h, w1, rstd, up[1])
        q8, s8, _ = ops.rms_norm_q8(o.reshape(B, N, D), w2, h)
        grads = [t.clone() for t in (dx, dk, dv, dw)]
        norm = ops.clip_grads_(grads, 0.1)
        return [o, dx, dk, dv, dw, q8.view(torch.uint8), s8, norm] + grads

    graphs = []
    for N, Nk in ((75, 190), (1, 3000)):          # (the second splits the keys)
        t, lens, H, up = together(60, torch.bfloat16, N, Nk)
        go(t, lens, H, up)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = go(t, lens, H, up)
        graphs.append((graph, t, lens, H, up, out, N, Nk))
    for seed in (61, 62, 63):
        for graph, t, lens, H, up, out, N, Nk in graphs:
            t2, lens2, _, up2 = together(seed, torch.bfloat16, N, Nk)
            for a, b in zip(t + list(up), t2 + list(up2)):
                a.copy_(b)
            lens.copy_(lens2.flip(0))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, t, lens, H, up, out, N, Nk in graphs:
            for a, b in zip(out, go(t, lens, H, up)):
                assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_backward_captured_while_an_eager_graph_of_the_same_leaves_lives():
    from ogmm_amd import train_ops
    if not ogmm_amd.graph_replay_safe():
        pytest.skip("the HIP runtime was initialised before graph packet capture could be switched off")
    tensors, lens, H, up = together(71, torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in tensors]

    def go():
        y, h = block(train_ops, leaves[0], leaves[1], leaves[2:4], leaves[4], leaves[5], H, kv_lens=lens)
        return y, h

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in torch.autograd.grad(go(), leaves, up)]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(go(), leaves, up)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_trainer_clips():
    """Trainer(max_grad_norm=): the step's gradients are un-scaled and clipped before Adam; far above the norm it is the un-clipped step, value for value"""
    from argparse import Namespace

    from ogmm_amd import synth
    from ogmm_amd.gmmreg import GMMReg
    from ogmm_amd.trainer import Trainer
    cfg = Namespace(gnn_k=20, num_heads=4, km_clusters=128, overlap_radius=0.035, n_clusters=16)
    B, N = 2, 256
    batch = synth.make_train_batch(0, B, N)
    batch = [b.cuda() for b in batch]
    starts = synth.fps_starts_for(0, B, N)
    got = {}
    for limit in (None, 1e9, 0.05):
        model = GMMReg(512, 16, cfg)
        synth.fill_state_dict(model.state_dict())
        trainer = Trainer(model.cuda(), lr=1e-4, welsch_top_k=64, max_grad_norm=limit)
        info = trainer.step(*batch, fps_starts=starts)
        assert not info["skipped"]
        got[limit] = ([p.grad.clone() for p in model.parameters() if p.grad is not None], [p.detach().clone() for p in model.parameters()], info)
    plain, wide, tight = got[None], got[1e9], got[0.05]
    assert "grad_norm" not in plain[2]
    total = math.sqrt(sum(float(t.double().square().sum()) for t in plain[0]))
    # (row scatter-adds of the step use atomics: two steps agree to their summation order, not bit for bit)
    assert abs(float(wide[2]["grad_norm"]) - total) <= 1e-4 * total
    assert abs(math.sqrt(sum(float(t.double().square().sum()) for t in tight[0])) - 0.05) <= 1e-6 and total > 0.05
    for a, b in zip(plain[1], wide[1]):
        assert float((a - b).abs().max()) <= 2.5e-4          # Adam's first step moves a value by the rate, whatever its gradient's size


# ---------------------------------------------------------------------------------------------- refusals (nothing is launched)
def test_refusals():
    from ogmm_amd import ops, train_ops
    from ogmm_amd._lib import OgmmError
    q, k, v, do = attention_case(2, 8, 12, 4, 2, 64, torch.bfloat16, 1)
    o, lse = ops.cross_attention(q, k, v, need_lse=True)
    mask = torch.ones(2, 12, dtype=torch.bool, device="cuda")
    bad = [
        lambda: ops.cross_attention(q, k.float(), v), lambda: ops.cross_attention(q, k[:, :, :1], v), lambda: ops.cross_attention(q[:1], k, v),
        lambda: ops.cross_attention(q[..., :60], k[..., :60], v[..., :60]), lambda: ops.cross_attention(q[:, :, :3], k, v), lambda: ops.cross_attention(q[0], k, v),
        lambda: ops.cross_attention(q.double(), k.double(), v.double()), lambda: ops.cross_attention(q, k, v, key_mask=mask.int()),
        lambda: ops.cross_attention(q, k, v, key_mask=mask[:, :5]), lambda: ops.cross_attention(q, k, v, kv_lens=torch.ones(2, device="cuda")),
        lambda: ops.cross_attention(q, k, v, kv_lens=torch.ones(3, dtype=torch.int32, device="cuda")), lambda: ops.cross_attention(q, k, v, q_lens=torch.ones(2, dtype=torch.int32)),
        lambda: ops.cross_attention(q, k.cpu(), v), lambda: ops.cross_attention(torch.cat([q] * 3, 3), torch.cat([k] * 3, 3), torch.cat([v] * 3, 3)),
        lambda: ops.cross_attention_bwd(q, k, v, o, lse, do[:, :4]), lambda: ops.cross_attention_bwd(q, k, v, o, lse, do.float()),
        lambda: ops.cross_attention_bwd(q, k, v, o.float(), lse, do), lambda: ops.cross_attention_bwd(q, k, v, o, lse[:, :1], do),
        lambda: train_ops.cross_attention(q, k, v[:, :5]), lambda: ops.cross_attention(q[..., :0], k[..., :0], v[..., :0])]
    x, w = randn(gen(1), 6, 40, dtype=torch.bfloat16), torch.ones(40, device="cuda")
    y, h, rstd = ops.rms_norm(x, w)
    bad += [
        lambda: ops.rms_norm(x, w[:39]), lambda: ops.rms_norm(x, w.half()), lambda: ops.rms_norm(x, w, x[:3]), lambda: ops.rms_norm(x, w, x.float()), lambda: ops.rms_norm(x.int(), w),
        lambda: ops.rms_norm(x, w, eps=-1.0), lambda: ops.rms_norm(x, w.cpu()), lambda: ops.rms_norm(torch.empty(1, 40000, device="cuda"), torch.empty(40000, device="cuda")),
        lambda: ops.rms_norm(x[:, :0], w[:0]), lambda: ops.rms_norm_q8(x, w, group=48), lambda: ops.rms_norm_q8(x, w, group=256), lambda: ops.rms_norm_bwd(y, h, w, rstd[:3]),
        lambda: ops.rms_norm_bwd(y.float(), h, w, rstd), lambda: ops.rms_norm_bwd(y, h, w, rstd, y[:2]), lambda: ops.rms_norm_bwd(y, h, w, rstd.double()), lambda: ops.rms_norm_bwd(y, h, w, rstd, residual=y[:3]),
        lambda: ops.rms_norm_bwd(y.float(), h.float(), w, rstd, residual=h.float())]
    a = torch.ones(100, device="cuda")
    bad += [
        lambda: ops.grad_norm([]), lambda: ops.clip_grads_([a, a], 1.0), lambda: ops.clip_grads_([a[:60], a[50:]], 1.0), lambda: ops.clip_grads_([a], -1.0), lambda: ops.clip_grads_([a], math.nan),
        lambda: ops.clip_grads_([a], 1.0, inv_scale=0.0), lambda: ops.clip_grads_([a], 1.0, inv_scale=math.inf), lambda: ops.clip_grads_([a.double()], 1.0), lambda: ops.clip_grads_([a[::2]], 1.0),
        lambda: ops.clip_grads_([a.expand(4, 100)], 1.0), lambda: ops.clip_grads_([a], 1.0, out=[]), lambda: ops.clip_grads_([a], 1.0, out=[a.half()]),
        lambda: ops.clip_grads_([a], 1.0, out=[a[:50]]), lambda: ops.clip_grads_([a[:50], a[50:]], 1.0, out=[a[50:], a[:50]]), lambda: ops.grad_norm([a, a.cpu()]),
        lambda: ops.clip_grads_([a.view(10, 10).t()], 1.0, out=[torch.empty(10, 10, device="cuda")])]
    for i, f in enumerate(bad):
        with pytest.raises(OgmmError):
            f()
            pytest.fail("call %d was not refused" % i)
    assert float(ops.clip_grads_([a[:50], a[50:]], 1e9, out=[a[:50], a[50:]])) > 0          # an output may be its own gradient
    torch.cuda.synchronize()
