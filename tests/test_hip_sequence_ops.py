"""GPU: cross attention, RMS norm and gradient clipping where values, rows or lists differ by orders of magnitude, where NaN and infinities stand, and at the sizes from which the
kernels take other routes; against plain evaluations in 64 bits.  The bounds count roundings as in test_hip_llm_ops.py."""
import math

import pytest
import torch

import ogmm_amd          # noqa: F401  (before anything touches the GPU: it switches the runtime's graph packet capture off)
from test_hip_llm_ops import IDS, TYPES, U, attention_case, check_attention, close, gen, half_step, randn

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- cross attention: gradients row by row
def heads(x):
    return x.double().permute(0, 2, 1, 3).contiguous()          # [B, heads, n, d]


def row_gradients(q, k, v, do):
    """{name: (gradient in 64 bits, bound of each row's error in the 2-norm)}, as many key heads as query heads, fp16.

    A row's error is a sum of roundings that know nothing of each other: it is held to four times the root of their squares' sum (each at its largest, h = 2^-11 of an operand).
    dS and P stand as fp16 operands at h, and not below 2^-38 of the bound that dS has over its query row (dq) or key (dk), |dO| |v| + |D|, 2^-39 for P.  Before that comes fp32: a score is d
    products (4 sqrt(d) roundings of its largest product), a row's weights have one sum over the keys in common.  The row sums D = dO o are formed from an o whose weights were rounded:
    P_ij e_D enters dS_ij."""
    B, Nq, H, d = q.shape
    Nk, h, a, c = k.shape[1], 2.0 ** -11, 2.0 ** -25, d ** -0.5
    Q, K, V, DO = map(heads, (q, k, v, do))

    def T(x):
        return x.transpose(2, 3).contiguous()

    def size(x):
        return (x * x).sum(dim=3, keepdim=True)

    S = Q @ T(K) * c
    r = U * (4 * math.sqrt(d) * float(Q.abs().max() * K.abs().max()) * c + 4 * math.sqrt(Nk) + 4 * float(S.abs().max()) + 32)
    P = torch.softmax(S, dim=3)
    dP = DO @ T(V)
    D = (P * dP).sum(dim=3, keepdim=True)
    dS = P * (dP - D)
    e_d = 4 * (h + r) * (P * dP).square().sum(dim=3, keepdim=True).sqrt()          # [.., Nq, 1]
    dq, dk, dv = dS @ K * c, T(dS) @ Q * c, T(P) @ DO
    e_ds = (h + r) * dS.abs()
    long_v, long_do = size(V).sqrt(), size(DO).sqrt()
    low_q = 2.0 ** -38 * (long_do * long_v.amax(dim=2, keepdim=True) + D.abs())
    low_k = 2.0 ** -38 * T(long_v * long_do.amax(dim=2, keepdim=True) + D.abs().amax(dim=2, keepdim=True))
    e_dq = 4 * c * ((e_ds + low_q).square() @ size(K)).sqrt() + c * e_d * size(P @ K).sqrt()
    e_dk = 4 * c * (T((e_ds + low_k).square() + (P * e_d).square()) @ size(Q)).sqrt()
    e_dv = 4 * (T(((h + r) * P + 2.0 ** -39).square()) @ size(DO)).sqrt()
    out = {}
    for name, x, e in (("dq", dq, e_dq), ("dk", dk, e_dk), ("dv", dv, e_dv)):
        out[name] = x.permute(0, 2, 1, 3), (e + (h + r) * size(x).sqrt() + a * math.sqrt(d)).permute(0, 2, 1, 3)[..., 0]
    return out


def check_row_gradients(q, k, v, do):
    from ogmm_amd import ops
    want = row_gradients(q, k, v, do)
    o, lse, rest = ops.cross_attention(q, k, v, need_lse=True, need_rest=True)
    for name, x in zip(("dq", "dk", "dv"), ops.cross_attention_bwd(q, k, v, o, lse, do, rest=rest)):
        off = (x.double() - want[name][0]).square().sum(dim=3).sqrt()
        bad = ~(off <= want[name][1])
        assert not bad.any(), "%s: %d of %d rows beyond the bound; worst off by %.3g of its size at a bound of %.3g" % (
            name, int(bad.sum()), bad.numel(), *(float((x / want[name][0].square().sum(dim=3).sqrt())[bad].max()) for x in (off, want[name][1])))


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("rows", ["one above the others", "half of them small", "each its own"])
def test_attention_fp16_rows_whose_gradients_differ(rows, d):
    """the gradient of a small row is its own, however large the others that share its key head are"""
    Nq, Nk = 256, 4096
    q, k, v, do = attention_case(1, Nq, Nk, 2, 1, d, torch.float16, 5 * d)
    if rows == "one above the others":
        by = torch.full((Nq,), 2.0 ** -6, device="cuda")
        by[77] = 2.0 ** 4
    elif rows == "half of them small":
        by = torch.where(torch.arange(Nq, device="cuda") % 2 == 0, 2.0 ** 0, 2.0 ** -7)
    else:
        by = 2.0 ** torch.arange(Nq, device="cuda").remainder(14).sub(7).float()
    check_row_gradients(q, k, v, (do.float() * by[None, :, None, None]).half())


@pytest.mark.parametrize("Nq,Nk,d", [(64, 400_001, 32), (33, 65_536, 128)])
def test_attention_fp16_gradients_of_many_keys(Nq, Nk, d):
    """weights of 1 / Nk each, far below fp16's normal numbers"""
    q, k, v, do = attention_case(1, Nq, Nk, 1, 1, d, torch.float16, Nk, size=0.3)
    check_row_gradients(q, k, v, do)


def test_attention_fp16_gradients_of_large_values():
    """values whose magnitudes add up to more than fp16 holds: dO v and dS leave its range, the gradients do not"""
    q, k, _, _ = attention_case(1, 50, 40, 1, 1, 128, torch.float16, 31, size=0.2)
    g = gen(32)
    sign = torch.where(torch.rand(128, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    v = (30000.0 * sign * torch.where(torch.arange(40, device="cuda") % 2 == 0, -1.0, 1.0)[:, None] * (0.5 + 0.5 * torch.rand(40, 128, generator=g, device="cuda"))).half()[None, :, None]
    do = (2.0 ** -12 * sign * (0.5 + torch.rand(50, 128, generator=g, device="cuda"))).half()[None, :, None]
    check_row_gradients(q, k, v, do)


# ---------------------------------------------------------------------------------------------- cross attention: NaN, infinities, rows that nobody has
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("Nq,G,Nk", [(5, 1, 90), (40, 1, 90), (200, 2, 300), (3, 4, 4000)])
def test_attention_rows_behind_their_lengths_beside_bad_keys(dtype, Nq, G, Nk):
    """rows behind q_lens give zeros (lse: -inf) in every output also where an admitted key or value is NaN or infinite"""
    from ogmm_amd import ops
    B, H, d = 2, 4, 64
    q, k, v, do = attention_case(B, Nq, Nk, H, G, d, dtype, 3)
    q_lens = torch.tensor([Nq // 2, 0], dtype=torch.int32, device="cuda")
    for at, what in ((k, math.nan), (v, math.nan), (v, math.inf), (k, -math.inf)):
        kept = at[:, 3].clone()
        at[:, 3] = what
        o, lse, rest = ops.cross_attention(q, k, v, q_lens=q_lens, need_lse=True, need_rest=True)
        dq, dk, dv = ops.cross_attention_bwd(q, k, v, o, lse, do, q_lens=q_lens, rest=rest)
        for b in range(B):
            n = int(q_lens[b])
            assert float(o[b, n:].abs().max()) == 0.0 and float(dq[b, n:].abs().max()) == 0.0 and bool((lse[b, :, n:] == -math.inf).all())
        assert float(dk[1].abs().max()) == 0.0 and float(dv[1].abs().max()) == 0.0          # (no row at all)
        at[:, 3] = kept


def test_attention_rows_behind_their_lengths_beside_bad_keys_with_more_scores_than_are_kept():
    from ogmm_amd import ops
    q, k, v, do = attention_case(1, 8200, 16400, 2, 2, 8, torch.float32, 11)
    q_lens = torch.tensor([8100], dtype=torch.int32, device="cuda")
    k[0, 5] = math.nan
    o, lse = ops.cross_attention(q, k, v, q_lens=q_lens, need_lse=True)
    dq, _, _ = ops.cross_attention_bwd(q, k, v, o, lse, do, q_lens=q_lens)
    assert float(dq[0, 8100:].abs().max()) == 0.0 and bool(torch.isnan(dq[0, :8100]).all())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("Nq,Nk", [(2, 1), (2, 100), (2, 5000), (70, 1), (70, 100), (70, 5000)])
def test_attention_of_a_nan_row(dtype, Nq, Nk):
    """a NaN query row looks at keys: its output and its log sum exp are NaN, not those of a row without a key; and so where every key is NaN"""
    from ogmm_amd import ops
    q, k, v, do = attention_case(1, Nq, Nk, 2, 1, 32, dtype, 8)
    good, lse_good = ops.cross_attention(q, k, v, need_lse=True)
    q2 = q.clone()
    q2[0, 1, 0] = math.nan
    o, lse = ops.cross_attention(q2, k, v, need_lse=True)
    assert bool(torch.isnan(o[0, 1, 0]).all()) and math.isnan(float(lse[0, 0, 1]))
    others = torch.ones(1, Nq, 2, dtype=torch.bool, device="cuda")
    others[0, 1, 0] = False
    # (a NaN makes its wave look for the other rows' maxima anew: their weights stand at another power, one more rounding each)
    assert float((o[others].double() - good[others].double()).norm()) <= 4 * (half_step(dtype) + 64 * U) * float(good[others].double().norm())
    assert bool(((lse - lse_good)[others.transpose(1, 2)].abs() <= 2 * (Nk + 64) * U + 8 * U * lse_good[others.transpose(1, 2)].abs()).all())
    dq, _, _ = ops.cross_attention_bwd(q2, k, v, o, lse, do)
    assert bool(torch.isnan(dq[0, 1, 0]).all()) and bool(torch.isfinite(dq[others]).all())
    o, lse = ops.cross_attention(q, k * math.nan, v, need_lse=True)
    assert bool(torch.isnan(o).all()) and bool(torch.isnan(lse).all())


# ---------------------------------------------------------------------------------------------- cross attention: sizes from which other routes are taken
@pytest.mark.parametrize("dtype,d", [(torch.float32, 32), (torch.float32, 24), (torch.bfloat16, 64), (torch.bfloat16, 40), (torch.float16, 64), (torch.float16, 16)])
@pytest.mark.parametrize("G", [1, 4])
def test_attention_many_rows_of_narrow_heads(dtype, d, G):
    """65536 rows and more of narrow heads: eight waves share a tile of keys"""
    B, Nq, Nk, H = 2, 8211, 333, 4
    q, k, v, do = attention_case(B, Nq, Nk, H, G, d, dtype, 6)
    kv_lens = torch.tensor([Nk, 190], dtype=torch.int32, device="cuda")
    q_lens = torch.tensor([8000, Nq], dtype=torch.int32, device="cuda")
    mask = torch.rand(B, Nk, generator=gen(7), device="cuda") < 0.8
    check_attention(q, k, v, do, grads=False)
    check_attention(q, k, v, do, grads=False, kv_lens=kv_lens, q_lens=q_lens, key_mask=mask)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_attention_of_many_batch_entries(dtype):
    """more than 64 entries of different lengths; and 64 of them, all alike but one"""
    B, Nq, Nk = 70, 40, 100
    q, k, v, do = attention_case(B, Nq, Nk, 2, 2, 32, dtype, 14)
    lens = torch.randint(0, Nk + 1, (B,), generator=gen(15), device="cuda", dtype=torch.int32)
    check_attention(q, k, v, do, kv_lens=lens)
    lens = torch.full((64,), 50, dtype=torch.int32, device="cuda")
    lens[63] = 77
    check_attention(q[:64], k[:64], v[:64], do[:64], kv_lens=lens)


def test_attention_gradient_offsets_past_31_bits():
    """the gradients of a cache of more than 2^31 elements: those of the last batch entry's keys stand where the keys do, all others are zero"""
    from ogmm_amd import ops
    B, Nk, Hkv, d, n = 17, 16384 * 8, 8, 128, 700          # 4.6 GB each for k, v and their gradients
    k = torch.zeros(B, Nk, Hkv, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    g = gen(2)
    for t in (k, v):
        t[-1, -n:] = randn(g, n, Hkv, d, dtype=torch.bfloat16)
    mask = torch.zeros(B, Nk, dtype=torch.bool, device="cuda")
    mask[-1, -n:] = True
    q, do = (randn(g, B, 1, 2 * Hkv, d, dtype=torch.bfloat16) for _ in range(2))
    o, lse = ops.cross_attention(q, k, v, key_mask=mask, need_lse=True)
    dq, dk, dv = ops.cross_attention_bwd(q, k, v, o, lse, do, key_mask=mask)
    short = [t[-1:, -n:].clone() for t in (k, v)]
    o1, lse1 = ops.cross_attention(q[-1:], *short, need_lse=True)
    want = ops.cross_attention_bwd(q[-1:], *short, o1, lse1, do[-1:])
    # (the two calls cut the keys differently: fp32 sums in another order, then one rounding each)
    for x, y in ((o[-1:], o1), (dq[-1:], want[0]), (dk[-1:, -n:], want[1]), (dv[-1:, -n:], want[2])):
        assert float((x.double() - y.double()).norm()) <= 2 * half_step(torch.bfloat16) * float(y.double().norm())
    assert float(dq[:-1].abs().max()) == 0.0
    for x in (dk, dv):
        assert not bool(x[-1, :-n].any()) and not any(bool(x[b].any()) for b in range(B - 1))


def test_attention_of_heads_far_apart():
    """256 heads that share a key head, 16 MB from one to the next: further than the kernels' 32 bits reach, so they are copied"""
    from ogmm_amd import ops
    q, k, v, do = attention_case(1, 3, 40, 256, 256, 8, torch.bfloat16, 23)
    far = torch.empty((1 << 31) + (1 << 23), dtype=torch.bfloat16, device="cuda").as_strided(q.shape, (8, 8, 1 << 23, 1))
    far.copy_(q)
    o, lse = ops.cross_attention(q, k, v, need_lse=True)
    assert torch.equal(ops.cross_attention(far, k, v), o)
    want = ops.cross_attention_bwd(q, k, v, o, lse, do)
    assert all(torch.equal(a, b) for a, b in zip(ops.cross_attention_bwd(far, k, v, o, lse, do), want))
    far.copy_(do)
    assert all(torch.equal(a, b) for a, b in zip(ops.cross_attention_bwd(q, k, v, o, lse, far), want))


def test_operators_called_by_threads_at_once():
    """four threads, each with a stream of its own, begin with the same calls at the same time: forward, gradient, norm and clipping are those of one thread"""
    import threading

    from ogmm_amd import ops
    cases = [attention_case(1, 70, 400, 4, 2, 128, t, i) for i, t in enumerate([torch.float32, torch.bfloat16, torch.float16, torch.bfloat16])]
    got, go = [None] * len(cases), threading.Barrier(len(cases))

    def work(i):
        q, k, v, do = cases[i]
        o, lse = ops.cross_attention(q, k, v, need_lse=True)
        dq, dk, dv = ops.cross_attention_bwd(q, k, v, o, lse, do)
        y, _, rstd = ops.rms_norm(dq, v[0, 0, 0])
        return [o, lse, dq, dk, dv, y, rstd, ops.clip_grads_([dk, dv], 0.5)]

    def thread(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            go.wait()
            got[i] = work(i)
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=thread, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(len(cases)):
        assert got[i] is not None and all(torch.equal(a, b) for a, b in zip(got[i], work(i)))


# ---------------------------------------------------------------------------------------------- RMS norm: rows that loop, magnitudes at the ends
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("R,D", [(140_001, 16), (70_003, 50), (20_001, 500), (5001, 2060), (1500, 8200), (1100, 16390)])
def test_norm_more_rows_than_workgroups(dtype, R, D):
    """every workgroup takes several rows, forward and backward: the first and the last rows and dw against 64 bits, and every row against a call of its own few"""
    from ogmm_amd import ops
    g = gen(R)
    x, r, dy, dh = (randn(g, R, D, dtype=dtype) for _ in range(4))
    w = (1 + 0.3 * randn(g, D)).to(dtype)
    y, h, rstd = ops.rms_norm(x, w, r)
    q, s, _ = ops.rms_norm_q8(x, w, r, group=128)
    back = (x, r) if dtype != torch.float32 else (h, None)
    dx, dw = ops.rms_norm_bwd(dy, back[0], w, rstd, dh, residual=back[1])
    dw64 = torch.zeros(D, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(dw64)
    step = 777          # rows of a call: one round of every shape
    for at in range(0, R, step):
        i = slice(at, at + step)
        y1, h1, rstd1 = ops.rms_norm(x[i], w, r[i])
        assert torch.equal(y[i], y1) and torch.equal(h[i], h1) and torch.equal(rstd[i], rstd1)
        q1, s1, _ = ops.rms_norm_q8(x[i], w, r[i], group=128)
        assert torch.equal(q[i].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[i], s1)
        few = slice(at, at + 100)          # (100 rows: one round of the backward)
        dx1, _ = ops.rms_norm_bwd(dy[few], back[0][few], w, rstd[few], dh[few], residual=None if back[1] is None else back[1][few])
        assert torch.equal(dx[few], dx1)
        H = x[i].double() + r[i].double() if dtype != torch.float32 else h[i].double()
        terms = dy[i].double() * H / ((H * H).mean(dim=1, keepdim=True) + 1e-6).sqrt()
        dw64 += terms.sum(dim=0)
        size += terms.abs().sum(dim=0)
    # as test_norm_gradient_from_the_summands
    close(dw, dw64, (64 + R // 64 + 48 + 41) * U * size + half_step(dtype) * dw64.abs() + 2.0 ** -25, "dw")
    assert torch.equal(ops.rms_norm_bwd(dy, back[0], w, rstd, dh, residual=back[1])[1], dw)


@pytest.mark.parametrize("dtype", TYPES[:2], ids=IDS.get)
@pytest.mark.parametrize("D", [5, 96, 500, 2000, 6000, 20000])
def test_norm_squares_outside_fp32(dtype, D):
    """rows whose squares, or their sum, leave fp32's range: the norm itself is inside it"""
    from ogmm_amd import ops
    g = gen(D)
    base, w = randn(g, 6, D), (1 + 0.3 * randn(g, D)).to(dtype)
    dy = randn(g, 6, D, dtype=dtype)
    sizes = torch.tensor([1e25, 1e-25, 1.0, 3e18, 1e30, 0.0], device="cuda")
    x = (base * sizes[:, None]).to(dtype)
    t, n = half_step(dtype), 48 * U
    for eps in (0.0, 1e-6, 1e-38):
        H = x.double()
        RS = 1 / ((H * H).mean(dim=1, keepdim=True) + eps).sqrt()
        live = [0, 1, 2, 3, 4] if eps == 0.0 else [0, 1, 2, 3, 4, 5]          # (a row of zeros without eps: 0 / 0)
        Y = H * RS * w.double()
        y, _, rstd = ops.rms_norm(x, w, eps=eps)
        close(y[live], Y[live], ((n + t) * Y.abs() + 2.0 ** -140)[live], "y")
        close(rstd[live], RS[live, 0], n * RS[live, 0], "rstd")
        assert eps > 0.0 or bool(torch.isnan(y[5]).all())
        q, s, _ = ops.rms_norm_q8(x, w, eps=eps)
        S = Y.abs().amax(dim=1, keepdim=True) / 448.0
        S = torch.where(S < 2.0 ** -126, torch.zeros_like(S), S)
        close(s[live], S[live], 2 * n * S[live], "scales")
        Q = q.double() * s.double()
        close(Q[live], torch.where(S == 0, torch.zeros_like(Y), Y)[live], (torch.maximum(2.0 ** -4 * Y.abs(), 2.0 ** -10 * S) * (1 + 2.0 ** -8) + 4 * n * Y.abs())[live], "q scales")
        if eps == 0.0:
            G, XH = dy.double() * w.double(), H * RS
            DX = RS * (G - XH * (G * XH).mean(dim=1, keepdim=True))
            size = RS * (G.abs() + XH.abs() * (G * XH).abs().mean(dim=1, keepdim=True))
            dx, _ = ops.rms_norm_bwd(dy[live], x[live], w, rstd[live])
            close(dx, DX[live], ((72 * U + 3 * n) * size + t * DX.abs() + 2.0 ** -134)[live], "dx")


@pytest.mark.parametrize("dtype", TYPES[:2], ids=IDS.get)
@pytest.mark.parametrize("D", [7, 300, 5000])
def test_norm_values_beside_the_largest_and_smallest(dtype, D):
    """values so large that times their weight they leave fp32, and rows so small that 1 / sqrt(mean(h^2)) does: y and its 8 bits are of ordinary size"""
    from ogmm_amd import ops
    g = gen(D)
    w = torch.full((D,), 3.0, device="cuda").to(dtype)
    x = torch.stack([s * (0.5 + 0.5 * torch.rand(D, generator=g, device="cuda")) for s in (3e38, 2.0 ** -130, -2e38)]).to(dtype)
    H = x.double()
    Y = H / (H * H).mean(dim=1, keepdim=True).sqrt() * 3.0
    t, n = half_step(dtype), 48 * U
    y, _, rstd = ops.rms_norm(x, w, eps=0.0)
    close(y, Y, (n + t) * Y.abs(), "y")
    q, s, _ = ops.rms_norm_q8(x, w, eps=0.0)
    S = Y.abs().amax(dim=1, keepdim=True) / 448.0
    close(s, S, 2 * n * S, "scales")
    close(q.double() * s.double(), Y, 2.0 ** -4 * (1 + 2.0 ** -8) * Y.abs() + 4 * n * Y.abs(), "q scales")


# ---------------------------------------------------------------------------------------------- gradients: lists of several runs, tensors in pieces, infinite limits
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("sizes", [[20_000_001, 15_000_003, 7, 9_000_000], [(1 << 30) + 5, 3]], ids=["runs", "pieces"])
def test_gradients_long_lists(dtype, sizes):
    """more values than one run a workgroup; a tensor longer than one entry of the kernels' table"""
    from ogmm_amd import ops
    g = gen(19)
    grads = [torch.empty(n, device="cuda", dtype=dtype).normal_(generator=g) for n in sizes]
    parts = [p for t in grads for p in t.split(1 << 26)]
    total = math.sqrt(sum(float(p.double().square().sum()) for p in parts))
    assert abs(float(ops.grad_norm(grads)) - total) <= 2 * U * total
    out = [torch.full(t.shape, math.nan, device="cuda") for t in grads]
    f = 3.0 / (total / 4 + 1e-6) / 4
    assert abs(float(ops.clip_grads_(grads, 3.0, inv_scale=0.25, out=out)) - total / 4) <= 2 * U * total / 4
    for p, o in zip(parts, [o for t in out for o in t.split(1 << 26)]):
        close(o, p.double() * f, 4 * U * p.double().abs() * f, "out")
    before = [p.clone() for p in parts]
    ops.clip_grads_(grads, 3.0, inv_scale=0.25)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for p, b in zip(parts, before):
        close(p, b.double() * f, (4 * U + half_step(dtype)) * b.double().abs() * f + tiny, "in place")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_gradients_infinite_norm_without_a_limit(dtype):
    """max_norm = inf un-scales and does nothing else, also where a gradient is infinite; a NaN still makes all of them NaN"""
    from ogmm_amd import ops
    a, b = torch.ones(5000, device="cuda", dtype=dtype), torch.full((33,), 8.0, device="cuda", dtype=dtype)
    a[17] = math.inf
    out = [torch.zeros(5000, device="cuda"), torch.zeros(33, device="cuda")]
    assert math.isinf(float(ops.clip_grads_([a, b], math.inf, inv_scale=0.25, out=out)))
    assert torch.equal(out[0], a.float() * 0.25) and torch.equal(out[1], b.float() * 0.25)
    assert math.isinf(float(ops.clip_grads_([a, b], math.inf, inv_scale=0.25)))
    assert torch.equal(a.float(), out[0]) and torch.equal(b.float(), out[1])
    a[18] = math.nan
    assert math.isnan(float(ops.clip_grads_([a, b], math.inf)))
    assert bool(torch.isnan(a).all()) and bool(torch.isnan(b).all())


# ---------------------------------------------------------------------------------------------- the trainer's gradients
@pytest.mark.parametrize("precision,loss_scale", [("f32", None), ("f32", 1024.0), ("f16x3", None)])
def test_trainer_clips_the_gradients_it_has(precision, loss_scale):
    """Trainer(max_grad_norm=): tensor by tensor the un-clipped step's gradients, times one factor where they are above the limit, with the loss scale taken out"""
    from argparse import Namespace

    from ogmm_amd import synth
    from ogmm_amd.gmmreg import GMMReg
    from ogmm_amd.trainer import Trainer
    cfg = Namespace(gnn_k=20, num_heads=4, km_clusters=128, overlap_radius=0.035, n_clusters=16, precision=precision)
    batch = [b.cuda() for b in synth.make_train_batch(0, 2, 256)]
    starts = synth.fps_starts_for(0, 2, 256)

    def gradients(limit):
        model = GMMReg(512, 16, cfg)
        synth.fill_state_dict(model.state_dict())
        trainer = Trainer(model.cuda(), welsch_top_k=64, loss_scale=loss_scale, max_grad_norm=limit)
        info = trainer.step(*batch, fps_starts=starts)
        assert not info["skipped"]
        return [None if p.grad is None else p.grad.double() for p in model.parameters()], info

    plain, _ = gradients(None)
    total = math.sqrt(sum(float(t.square().sum()) for t in plain if t is not None))
    for limit in (1e9, math.inf, 0.05 * total):
        got, info = gradients(limit)
        factor = min(1.0, limit / (total + 1e-6))
        # (row scatter-adds of the step use atomics: two steps agree to their summation order, 1e-4 of the whole)
        assert abs(float(info["grad_norm"]) - total) <= 1e-4 * total
        far = 0.0
        for a, b in zip(got, plain):
            assert (a is None) == (b is None)
            if a is not None:
                assert bool(a.any()) == bool(b.any())
                far += float((a - factor * b).square().sum())
        assert math.sqrt(far) <= 2e-4 * factor * total
