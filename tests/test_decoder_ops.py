"""Cross attention, token embeddings and the orthogonalised optimiser step against float64.

Tolerances come from the arithmetic, u = 2^-24 (half a step of fp32).  A sum of n rounded terms is off by
at most LAM * sqrt(n) * u times the sum of their magnitudes, but for a chance of 2 exp(-LAM^2 / 2) (rounding
errors as independent, mean-zero variables); LAM = 6 makes that 3e-8.  The helpers below carry that
through softmax and its gradient element by element, so the bound of every element is its own.
"""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

U = 2.0 ** -24
LAM = 6.0
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from visiontransformer_amd import vitk
    vitk.init(0)
    return vitk


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def within(got, want, tol, what=""):
    got, want = got.double().cpu(), want.cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - tol.cpu()
    worst = over.argmax()
    assert (over <= 0).all(), (f"{what}: element {int(worst)} of {tuple(got.shape)} is {got.flatten()[worst].item()}, expected "
                               f"{want.flatten()[worst].item()} +- {tol.cpu().expand_as(want).flatten()[worst].item()}")


# ------------------------------------------------------------------------------- cross attention
def attention64(q, k, v, lens, scale, dout=None):
    """float64 out (dq, dk, dv) and the bound of each element of each, one (batch, head) at a time."""
    B, Nq, H, dh = q.shape
    Nk, Hkv = k.shape[1:3]
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    res = {n: torch.zeros_like(x) for n, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    tol = {n: torch.zeros_like(x) for n, x in res.items()}
    stats = torch.zeros(B, H, Nq, 2, dtype=torch.float64)
    root = lambda n: LAM * np.sqrt(n) * U  # noqa: E731
    for b in range(B):
        n = Nk if lens is None else min(max(int(lens[b]), 0), Nk)
        if n == 0:
            continue
        for h in range(H):
            j = h // (H // Hkv)
            Q, Kk, Vv = q[b, :, h], k[b, :n, j], v[b, :n, j]
            s = scale * Q @ Kk.T
            m = s.amax(1, keepdim=True)
            e = torch.exp(s - m)
            l = e.sum(1, keepdim=True)
            p = e / l
            out = p @ Vv
            res["out"][b, :, h] = out
            stats[b, h, :, 0], stats[b, h, :, 1] = m[:, 0], l[:, 0]
            # score: a dot of dh terms, the product with scale log2 e (2 roundings, of s and of the maximum)
            es = root(dh) * abs(scale) * (Q.abs() @ Kk.abs().T) + 4 * U * (s.abs() + m.abs())
            # probability, relative: exponent errors of the key and of the maximum's stand-in, exp2 (2 u), sum, 1/l
            rel = es + (p * es).sum(1, keepdim=True) + (root(n) + 8 * U)
            ep = p * rel
            eo = ep @ Vv.abs() + root(n) * (p @ Vv.abs()) + 2 * U * out.abs()
            tol["out"][b, :, h] = eo
            if dout is None:
                continue
            G = dout[b, :, h].double().cpu()
            dp = G @ Vv.T
            delta = (G * out).sum(1, keepdim=True)
            ds = p * (dp - delta)
            edp = root(dh) * (G.abs() @ Vv.abs().T)
            edl = (G.abs() * eo).sum(1, keepdim=True) + root(dh) * (G.abs() * out.abs()).sum(1, keepdim=True)
            eds = p * (edp + edl + 2 * U * (dp.abs() + delta.abs())) + ep * (dp - delta).abs()
            res["dq"][b, :, h] = scale * ds @ Kk
            tol["dq"][b, :, h] = abs(scale) * (eds @ Kk.abs() + (root(n) + 2 * U) * (ds.abs() @ Kk.abs()))
            res["dk"][b, :n, j] += scale * ds.T @ Q
            # rows of all heads of the group go into one sum
            r = root(Nq * (H // Hkv)) + 2 * U
            tol["dk"][b, :n, j] += abs(scale) * (eds.T @ Q.abs() + r * (ds.abs().T @ Q.abs()))
            res["dv"][b, :n, j] += p.T @ G
            tol["dv"][b, :n, j] += ep.T @ G.abs() + r * (p.T @ G.abs())
    return res, tol, stats


def pitched(g, B, N, heads, dh, pad, offset=0):
    """[B, N, heads, dh] inside rows of heads*dh + pad floats, `offset` floats into the allocation."""
    flat = randn(g, B * N * (heads * dh + pad) + offset)[offset:]
    return flat.reshape(B, N, heads * dh + pad)[:, :, :heads * dh].unflatten(2, (heads, dh))


ATTENTION = {
    # B, H, Hkv, Nq, Nk, dh, lengths, row padding, offset
    "one_by_one": (1, 1, 1, 1, 1, 1, None, 0, 0),
    "token_over_197": (4, 12, 12, 1, 197, 64, None, 0, 0),
    "token_shared_heads_long": (3, 8, 2, 1, 5001, 128, [5001, 0, 1234], 0, 0),
    "token_three_rows_dh_24": (2, 6, 2, 1, 700, 24, [700, 3], 0, 0),
    "few_rows_of_two_tokens": (2, 8, 4, 3, 129, 96, [0, 129], 4, 0),
    "eight_rows_split": (1, 8, 1, 1, 4000, 128, None, 0, 0),
    "many_heads_no_split": (48, 12, 12, 1, 1500, 32, None, 0, 0),
    "nine_rows": (2, 9, 1, 1, 2100, 64, [2100, 65], 0, 0),
    "token_all_heads_share_one": (2, 7, 1, 1, 333, 48, [1, 332], 4, 0),
    "prompt": (2, 3, 3, 33, 197, 64, None, 0, 0),
    "one_key": (3, 4, 4, 70, 1, 64, None, 0, 0),
    "ragged": (5, 6, 6, 65, 130, 32, [130, 0, 1, 129, 64], 0, 0),
    "lengths_outside": (3, 2, 2, 9, 40, 64, [-5, 41, 2 ** 31 - 1], 0, 0),
    "odd_dh_unaligned": (2, 3, 1, 37, 75, 33, [75, 31], 1, 1),
    "dh_96_shared": (2, 8, 2, 130, 261, 96, [200, 261], 0, 0),
    "dh_128_masked": (1, 2, 2, 257, 129, 128, None, 4, 4),
    "dh_7": (2, 5, 5, 17, 19, 7, None, 0, 0),
    "few_keys_many_rows": (2, 6, 6, 147, 50, 64, None, 0, 0),
    "long_keys_split": (1, 2, 1, 40, 3001, 64, [2999], 0, 0),
    "long_rows": (1, 2, 1, 1500, 70, 80, None, 0, 0),
    # all keys of a head in one workgroup of the backward: rows of shared heads, split; lengths; alignment
    "few_keys_shared_split": (3, 6, 2, 333, 64, 64, [64, 0, 33], 0, 0),
    "few_keys_narrow": (2, 4, 1, 700, 31, 32, [31, 16], 4, 0),
    "few_keys_unaligned": (2, 3, 1, 95, 49, 35, [49, 17], 1, 1),
    "one_key_many_rows": (2, 2, 2, 1000, 1, 8, None, 0, 0),
    "few_keys_full_device": (64, 8, 8, 45, 40, 60, None, 4, 0),
    # single tokens: more than 64 parts, lengths far below the longest, more heads than CUs
    "token_many_parts": (1, 2, 1, 1, 30011, 72, None, 0, 0),
    "token_many_parts_ragged": (3, 4, 1, 1, 20000, 40, [20000, 3, 70], 0, 0),
    "token_heads_over_cus": (70, 8, 8, 1, 130, 20, [130 - b for b in range(70)], 0, 0),
}


@gpu
@pytest.mark.parametrize("name", list(ATTENTION))
def test_cross_attention_forward_and_backward(K, name):
    B, H, Hkv, Nq, Nk, dh, lens, pad, off = ATTENTION[name]
    g = rng(100 + list(ATTENTION).index(name))
    q, k, v = (pitched(g, B, n, h, dh, pad, off) for n, h in ((Nq, H), (Nk, Hkv), (Nk, Hkv)))
    dout = pitched(g, B, Nq, H, dh, pad, off)
    out, dq = torch.full_like(q, 7.0), pitched(g, B, Nq, H, dh, pad, off)
    dk, dv = (pitched(g, B, Nk, Hkv, dh, pad, off) for _ in range(2))
    klen = None
    if lens is not None:
        klen = torch.tensor(lens, dtype=torch.int32, device="cuda")
        for b, n in enumerate(lens):  # what lies behind a length is never read
            k[b, max(n, 0):] = float("nan")
            v[b, max(n, 0):] = float("nan")
    stats = torch.full((B * H, Nq, 2), 7.0, device="cuda")
    want, tol, wstats = attention64(q, k.nan_to_num(), v.nan_to_num(), lens, dh ** -0.5, dout)
    args = K.cross_sdpa_args(q, k, v, out, key_len=klen, stats=stats, dout=dout, dq=dq, dk=dk, dv=dv)
    K.cross_sdpa_fwd(args)
    within(out, want["out"], tol["out"], "out")
    got = stats.double().cpu().view(B, H, Nq, 2)
    m = got[..., 0] / np.log2(np.e)
    assert ((m - wstats[..., 0]).abs() <= 1e-5 * (1 + wstats[..., 0].abs())).all()
    assert ((got[..., 1] - wstats[..., 1]).abs() <= 1e-4 * (1 + wstats[..., 1])).all()
    K.cross_sdpa_bwd(args)
    for n, t in (("dq", dq), ("dk", dk), ("dv", dv)):
        within(t, want[n], tol[n], n)
    # same bits again, and without statistics
    first = [t.clone() for t in (out, dq, dk, dv)]
    K.cross_sdpa_fwd(args)
    K.cross_sdpa_bwd(args)
    for a, b in zip(first, (out, dq, dk, dv)):
        assert torch.equal(a, b)
    out2 = torch.full_like(q, 7.0)
    K.cross_sdpa_fwd(K.cross_sdpa_args(q, k, v, out2, key_len=klen))
    assert torch.equal(out2, out)


@gpu
@pytest.mark.parametrize("dh", [20, 64, 88, 128])
def test_cross_attention_every_block_size(K, dh):
    """Rows and keys of each count of 16-row groups (2, 4, 8, more than one block) against each other."""
    for Nq in (17, 40, 100, 131):
        for Nk in (13, 33, 70, 140):
            g = rng(1000 * Nq + Nk)
            q, k, v, dout = randn(g, 2, Nq, 2, dh), randn(g, 2, Nk, 2, dh), randn(g, 2, Nk, 2, dh), randn(g, 2, Nq, 2, dh)
            lens = [Nk, Nk - 7]
            want, tol, _ = attention64(q, k, v, lens, dh ** -0.5, dout)
            out, dq, dk, dv = (torch.full_like(x, 7.0) for x in (q, q, k, v))
            a = K.cross_sdpa_args(q, k, v, out, key_len=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                  stats=torch.empty(4, Nq, 2, device="cuda"), dout=dout, dq=dq, dk=dk, dv=dv)
            K.cross_sdpa_fwd(a)
            K.cross_sdpa_bwd(a)
            for n, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
                within(t, want[n], tol[n], f"{n} {Nq} x {Nk}")


@gpu
@pytest.mark.parametrize("dh", [20, 64, 88, 128])
def test_cross_attention_every_block_size_with_many_heads(K, dh):
    """Blocks of 64 as four waves, which at least one workgroup a CU takes: alone, as 3 and 5 blocks, over keys of
    every kind of count."""
    for Nq, Nk in ((40, 33), (60, 130), (131, 50), (190, 200), (120, 64), (259, 20), (20, 150), (140, 300)):
        g = rng(1000 * Nq + Nk)
        B, Hkv = 40, 8  # 320 workgroups
        q, k, v, dout = (randn(g, B, n, Hkv, dh) for n in (Nq, Nk, Nk, Nq))
        lens = [Nk - b if b % 8 else Nk for b in range(B)]
        lens[3] = 0
        want, tol, _ = attention64(q, k, v, lens, dh ** -0.5, dout)
        out, dq, dk, dv = (torch.full_like(x, 7.0) for x in (q, q, k, v))
        a = K.cross_sdpa_args(q, k, v, out, key_len=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                              stats=torch.empty(B * Hkv, Nq, 2, device="cuda"), dout=dout, dq=dq, dk=dk, dv=dv)
        K.cross_sdpa_fwd(a)
        K.cross_sdpa_bwd(a)
        for n, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
            within(t, want[n], tol[n], f"{n} {Nq} x {Nk}")


@gpu
@pytest.mark.parametrize("dh", [8, 60, 100])
def test_cross_attention_few_rows_of_every_count(K, dh):
    for rows in range(1, 9):
        for Nk in (3, 300, 2500):  # one launch of sixteen waves; split and joined
            g = rng(10 * rows + Nk)
            q, k, v = randn(g, 2, 1, rows, dh), randn(g, 2, Nk, 1, dh), randn(g, 2, Nk, 1, dh)
            lens = [Nk - 2, Nk]
            want, tol, wst = attention64(q, k, v, lens, -dh ** -0.5)
            out, st = torch.full_like(q, 7.0), torch.empty(2 * rows, 1, 2, device="cuda")
            K.cross_sdpa_fwd(K.cross_sdpa_args(q, k, v, out, key_len=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                               stats=st, scale=-dh ** -0.5))
            within(out, want["out"], tol["out"], f"{rows} rows, {Nk} keys")
            l = st.double().cpu().view(2, rows, 1, 2)[..., 1]
            assert ((l - wst[..., 1]).abs() <= 1e-4 * (1 + wst[..., 1])).all()


@gpu
def test_cross_attention_splits_where_blocks_are_few(K):
    """The forms with parts really run at the sizes that the tests above use for them."""
    def need(fn, **kw):
        return fn(C.byref(_xargs(K, **kw)))
    d = K.dll()
    long_keys = dict(B=1, H=2, Hkv=1, Nq=40, Nk=3001, dh=64, ld_q=128, ld_k=64, ld_v=64, ld_out=128, ld_dout=128, ld_dq=128,
                     ld_dk=64, ld_dv=64)
    assert need(d.vitk_cross_sdpa_fwd_workspace_bytes, **long_keys) > 0
    assert need(d.vitk_cross_sdpa_bwd_workspace_bytes, **long_keys) > 4096
    long_rows = dict(long_keys, Nq=1500, Nk=70)
    assert need(d.vitk_cross_sdpa_bwd_workspace_bytes, **long_rows) > 4 * 2 * 1500 + 4096


@gpu
@pytest.mark.parametrize("cus", [8, 64, 1024])
def test_cross_attention_on_the_routes_of_other_devices(K, cus):
    """Kernels, blocks and splits follow the number of CUs; every one of them is right for every size."""
    shapes = ((2, 4, 2, 1, 500, 64), (3, 8, 8, 1, 2000, 128), (2, 8, 4, 3, 700, 80), (4, 4, 4, 20, 300, 64),
              (4, 8, 8, 40, 100, 64), (2, 4, 2, 70, 330, 96), (1, 2, 2, 300, 500, 128), (5, 6, 6, 147, 50, 32),
              (1, 1, 1, 9, 2000, 33))
    K.planning_cu_count(cus)
    try:
        for B, H, Hkv, Nq, Nk, dh in shapes:
            g = rng(Nq + Nk + dh)
            q, dout = randn(g, B, Nq, H, dh), randn(g, B, Nq, H, dh)
            k, v = randn(g, B, Nk, Hkv, dh), randn(g, B, Nk, Hkv, dh)
            lens = [Nk - 13 * b for b in range(B)]
            want, tol, _ = attention64(q, k, v, lens, dh ** -0.5, dout)
            out, dq, dk, dv = (torch.full_like(x, 7.0) for x in (q, q, k, v))
            a = K.cross_sdpa_args(q, k, v, out, key_len=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                  stats=torch.empty(B * H, Nq, 2, device="cuda"), dout=dout, dq=dq, dk=dk, dv=dv)
            K.cross_sdpa_fwd(a)
            K.cross_sdpa_bwd(a)
            for n, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
                within(t, want[n], tol[n], f"{n} {Nq} x {Nk} x {dh}")
    finally:
        K.planning_cu_count(0)


@gpu
def test_cross_attention_leaves_what_is_between_the_rows(K):
    g = rng(5)
    B, H, N, dh = 2, 3, 11, 20
    bufs = {n: torch.full((B, N + (n[-1] in "kv") * 8, H * dh + 12), 3.0, device="cuda") for n in ("out", "dq", "dk", "dv")}
    view = {n: t[:, :, :H * dh].unflatten(2, (H, dh)) for n, t in bufs.items()}
    q, k, v, dout = randn(g, B, N, H, dh), randn(g, B, N + 8, H, dh), randn(g, B, N + 8, H, dh), randn(g, B, N, H, dh)
    stats = torch.empty(B * H, N, 2, device="cuda")
    args = K.cross_sdpa_args(q, k, v, view["out"], stats=stats, dout=dout, dq=view["dq"], dk=view["dk"], dv=view["dv"])
    K.cross_sdpa_fwd(args)
    K.cross_sdpa_bwd(args)
    for n, t in bufs.items():
        assert (t[:, :, H * dh:] == 3.0).all(), n
        assert (t[:, :, :H * dh] != 3.0).all(), n


@gpu
def test_cross_attention_without_queries_or_keys(K):
    B, H, dh = 2, 3, 16
    g = rng(6)
    e = lambda n: torch.full((B, n, H, dh), 7.0, device="cuda")  # noqa: E731
    # no keys: zeros out, zero gradient
    out, dq, st = e(5), e(5), torch.full((B * H, 5, 2), 7.0, device="cuda")
    a = K.cross_sdpa_args(randn(g, B, 5, H, dh), e(0), e(0), out, stats=st, dout=e(5), dq=dq, dk=e(0), dv=e(0))
    K.cross_sdpa_fwd(a)
    K.cross_sdpa_bwd(a)
    assert (out == 0).all() and (st == 0).all() and (dq == 0).all()
    # no queries: the key gradients are zeros
    dk, dv = e(6), e(6)
    st = torch.empty(B * H, 0, 2, device="cuda")
    a = K.cross_sdpa_args(e(0), e(6), e(6), e(0), stats=st, dout=e(0), dq=e(0), dk=dk, dv=dv)
    K.cross_sdpa_fwd(a)
    K.cross_sdpa_bwd(a)
    assert (dk == 0).all() and (dv == 0).all()


@gpu
@pytest.mark.parametrize("amplitude", [1e-18, 30.0])
def test_cross_attention_extreme_scores(K, amplitude):
    """Scores that underflow to one uniform row, and scores in the thousands (one key takes all)."""
    g = rng(7)
    B, H, Nq, Nk, dh = 1, 2, 40, 300, 64
    q, k = randn(g, B, Nq, H, dh) * amplitude, randn(g, B, Nk, H, dh) * amplitude
    v, dout = randn(g, B, Nk, H, dh), randn(g, B, Nq, H, dh) * 1e-6
    want, tol, _ = attention64(q, k, v, None, dh ** -0.5, dout)
    out, dq, dk, dv = (torch.empty_like(x) for x in (q, q, k, v))
    stats = torch.empty(B * H, Nq, 2, device="cuda")
    a = K.cross_sdpa_args(q, k, v, out, stats=stats, dout=dout, dq=dq, dk=dk, dv=dv)
    K.cross_sdpa_fwd(a)
    K.cross_sdpa_bwd(a)
    tiny = 2.0 ** -126  # subnormal results may be flushed
    for n, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        within(t, want[n], tol[n] + tiny, n)


@gpu
@pytest.mark.parametrize("Nq, Nk, dh", [(1, 197, 64), (2, 40, 128), (40, 197, 64), (150, 500, 96), (70, 50, 32)])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_cross_attention_keeps_what_is_not_finite_to_its_own(K, Nq, Nk, dh, value):
    """An infinity or NaN reaches the results that are formed from it and no others: those keep their bits."""
    g, B, H, Hkv = rng(380), 2, 4, 2
    q, k, v, dout = randn(g, B, Nq, H, dh), randn(g, B, Nk, Hkv, dh), randn(g, B, Nk, Hkv, dh), randn(g, B, Nq, H, dh)
    inputs = dict(q=q, k=k, v=v, dout=dout)
    names = ("out", "dq", "dk", "dv")

    def run():
        o, dq, dk, dv = (torch.full_like(t, 7.0) for t in (q, q, k, v))
        args = K.cross_sdpa_args(q, k, v, o, stats=torch.empty(B * H, Nq, 2, device="cuda"), dout=dout, dq=dq, dk=dk, dv=dv)
        K.cross_sdpa_fwd(args)
        K.cross_sdpa_bwd(args)
        return dict(zip(names, (o, dq, dk, dv)))

    clean = run()
    row, key, col = Nq - 1, Nk // 2, dh // 2
    all_ = slice(None)
    # the element of each input, and what is formed from it: (batch, token, heads, column) of each result
    head = dict(q=(1, row, 3, col), dout=(1, row, 3, col), k=(1, key, 1, col), v=(1, key, 1, col))
    reach = {
        "q": dict(out=(1, row, 3), dq=(1, row, 3), dk=(1, all_, 1), dv=(1, all_, 1)),
        "dout": dict(dq=(1, row, 3), dk=(1, all_, 1), dv=(1, all_, 1)),
        "k": dict(out=(1, all_, slice(2, 4)), dq=(1, all_, slice(2, 4)), dk=(1, all_, 1), dv=(1, all_, 1)),
        "v": dict(out=(1, all_, slice(2, 4), col), dq=(1, all_, slice(2, 4)), dk=(1, all_, 1)),
    }
    for name, x in inputs.items():
        old = x[head[name]].clone()
        x[head[name]] = value
        got = run()
        x[head[name]] = old
        for n in names:
            same = torch.ones_like(got[n], dtype=torch.bool)
            if n in reach[name]:
                same[reach[name][n]] = False
            assert torch.equal(got[n][same], clean[n][same]), (name, n)
        if value != value:  # NaN stays NaN
            assert name not in ("q", "k") or torch.isnan(got["out"][1, row, 3]).all(), name
            assert name not in ("k", "v") or torch.isnan(got["out"][1, :, 2:4, col]).all(), name
            assert torch.isnan(got["dq"][1, row, 3]).all(), name
        if name == "v" and abs(value) == float("inf"):  # every probability is above 0 here
            assert not torch.isfinite(got["out"][1, :, 2:4, col]).any()


def check_attention(K, q, k, v, lens, scale, dout, like=torch.empty_like):
    """Forward, statistics and gradients of one call against attention64."""
    B, Nq, H, dh = q.shape
    out, dq, dk, dv = (like(t).fill_(7.0) for t in (q, q, k, v))
    stats = torch.empty(B * H, Nq, 2, device="cuda")
    klen = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    args = K.cross_sdpa_args(q, k, v, out, key_len=klen, scale=scale, stats=stats, dout=dout, dq=dq, dk=dk, dv=dv)
    K.cross_sdpa_fwd(args)
    K.cross_sdpa_bwd(args)
    want, tol, _ = attention64(q, k, v, lens, scale, dout)
    for name, got in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        within(got, want[name], tol[name] + 1e-30, name)


@gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, -2.0])
@pytest.mark.parametrize("Nq, Nk, dh", [(1, 197, 64), (37, 40, 64), (40, 150, 96), (5, 2100, 32)])
def test_cross_attention_scales_of_any_sign(K, scale, Nq, Nk, dh):
    g = rng(390)
    q, dout = randn(g, 2, Nq, 4, dh), randn(g, 2, Nq, 4, dh)
    k, v = randn(g, 2, Nk, 2, dh) * 0.5, randn(g, 2, Nk, 2, dh)
    check_attention(K, q, k, v, [Nk, Nk // 2], scale, dout)


@gpu
@pytest.mark.parametrize("Nq, Nk", [(1, 90), (20, 90), (20, 40), (130, 70)])
def test_cross_attention_ragged_batches_of_more_than_a_wave(K, Nq, Nk):
    g, B = rng(391), 70
    lens = [(17 * b) % (Nk + 1) for b in range(B)]
    q, dout, k, v = randn(g, B, Nq, 2, 16), randn(g, B, Nq, 2, 16), randn(g, B, Nk, 1, 16), randn(g, B, Nk, 1, 16)
    check_attention(K, q, k, v, lens, 0.25, dout)


@gpu
@pytest.mark.parametrize("Nq, Nk, dh", [(1, 1100, 64), (1100, 70, 32), (33, 1100, 64), (1100, 9, 64)])
def test_cross_attention_offsets_past_32_bits(K, Nq, Nk, dh):
    """Rows 2^21 floats apart: the last ones lie more than 2^31 elements behind the first."""
    g, H, ld = rng(392), 2, 2 ** 21
    need = max(Nq, Nk) * ld
    assert need > 2 ** 31
    room = torch.empty(need, device="cuda")
    place = [0]

    def far(t):  # rows of all tensors lie side by side
        B, N, heads, d = t.shape
        r = room.as_strided((B, N, heads, d), (N * ld, ld, d, 1), place[0])
        place[0] += heads * d
        return r.copy_(t)

    q, dout, k, v = (far(randn(g, 1, n, H, dh)) for n in (Nq, Nq, Nk, Nk))
    check_attention(K, q, k, v, None, 0.2, dout, like=lambda t: far(torch.zeros(t.shape, device="cuda")))


@gpu
def test_cross_attention_gradients_against_differences(K):
    """Central differences of sum(out * dout) in float64 of the definition, at single entries."""
    g = rng(8)
    B, H, Hkv, Nq, Nk, dh = 2, 4, 2, 5, 9, 12
    q, k, v, dout = randn(g, B, Nq, H, dh), randn(g, B, Nk, Hkv, dh), randn(g, B, Nk, Hkv, dh), randn(g, B, Nq, H, dh)
    lens = [9, 4]
    out, dq, dk, dv = (torch.empty_like(x) for x in (q, q, k, v))
    stats = torch.empty(B * H, Nq, 2, device="cuda")
    a = K.cross_sdpa_args(q, k, v, out, key_len=torch.tensor(lens, dtype=torch.int32, device="cuda"), stats=stats, dout=dout,
                          dq=dq, dk=dk, dv=dv)
    K.cross_sdpa_fwd(a)
    K.cross_sdpa_bwd(a)
    base = {"q": q.double().cpu(), "k": k.double().cpu(), "v": v.double().cpu()}
    G = dout.double().cpu()

    def f(**kw):
        x = dict(base, **kw)
        o = torch.zeros_like(x["q"])
        for b in range(B):
            for h in range(H):
                n, j = lens[b], h // 2
                p = torch.softmax(dh ** -0.5 * x["q"][b, :, h] @ x["k"][b, :n, j].T, 1)
                o[b, :, h] = p @ x["v"][b, :n, j]
        return (o * G).sum().item()

    step = 1e-5
    for n, t in (("q", dq), ("k", dk), ("v", dv)):
        for at in ((0, 1, 1, 3), (1, 3, 0, 0), (1, 4, 1, 7)):
            plus, minus = base[n].clone(), base[n].clone()
            plus[at] += step
            minus[at] -= step
            d = (f(**{n: plus}) - f(**{n: minus})) / (2 * step)
            # differences: 1e-10 of the third derivative, 1e-11 / step of rounding; the kernel: about 1e-6
            assert abs(t[at].item() - d) <= 2e-5 * (1 + abs(d)), (n, at)


@gpu
def test_cross_attention_captured_and_replayed_on_another_stream(K):
    """Forward and backward in one graph, replayed with other inputs and lengths, eager work between."""
    g = rng(9)
    B, H, Hkv, Nq, Nk, dh = 2, 4, 2, 1, 2000, 64
    q, k, v, dout = randn(g, B, Nq, H, dh), randn(g, B, Nk, Hkv, dh), randn(g, B, Nk, Hkv, dh), randn(g, B, Nq, H, dh)
    klen = torch.tensor([Nk, 7], dtype=torch.int32, device="cuda")
    mk = lambda: [torch.full_like(x, 7.0) for x in (q, q, k, v)]  # noqa: E731
    (out, dq, dk, dv), eager = mk(), mk()
    stats = [torch.empty(B * H, Nq, 2, device="cuda") for _ in range(2)]
    a = K.cross_sdpa_args(q, k, v, out, key_len=klen, stats=stats[0], dout=dout, dq=dq, dk=dk, dv=dv)
    e = K.cross_sdpa_args(q, k, v, eager[0], key_len=klen, stats=stats[1], dout=dout, dq=eager[1], dk=eager[2], dv=eager[3])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        K.cross_sdpa_fwd(a)
        K.cross_sdpa_bwd(a)
    for i in range(4):
        q.copy_(randn(g, *q.shape))
        v.copy_(randn(g, *v.shape))
        klen.copy_(torch.tensor([i * 600, Nk - i], dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        K.cross_sdpa_fwd(e)
        K.cross_sdpa_bwd(e)
        torch.cuda.synchronize()
        for x, y in zip((out, dq, dk, dv), eager):
            assert torch.equal(x, y), i


# ---------------------------------------------------------------------------------- embeddings
EMBED = {
    # V, D, rows, how the tokens are drawn
    "one": (1, 1, 1, "uniform"),
    "odd_width": (37, 33, 100, "uniform"),
    "wide": (1000, 768, 528, "rank"),
    "one_token_takes_all": (500, 192, 5000, "same"),
    "padded": (300, 500, 1111, "padded"),
    "all_padding": (64, 64, 77, "all_padding"),
    "outside": (100, 96, 400, "outside"),
    "many_tokens": (5000, 96, 70001, "rank"),
    "few_tokens_one_takes_most": (40, 300, 1023, "same"),
    "sorted_small_table": (7, 64, 1025, "uniform"),
    "sorted_few_tokens": (4097, 260, 65, "padded"),
    "one_chunk": (5000, 48, 32, "rank"),
    "three_passes": (70001, 36, 3000, "rank"),
    "one_token_takes_all_long": (5000, 20, 200003, "same"),
    "two_levels": (20000, 12, 40000, "rank"),
    "large_table_few_tokens": (100003, 32, 9, "uniform"),
    # placed by counting (up to 8192 tokens; 4096 over a table of one digit), by digits behind that
    "counted_most": (20000, 40, 8192, "rank"),
    "counted_odd": (70001, 36, 8191, "padded"),
    "counted_outside": (20000, 32, 3333, "outside"),
    "counted_one_chunk": (20000, 48, 31, "rank"),
    "counted_small_table": (200, 64, 4096, "rank"),
    "digits_two": (3000, 64, 8193, "rank"),
    "digits_one": (200, 64, 4097, "padded"),
    "digits_three": (70001, 36, 9001, "rank"),
    "direct_largest_table": (16384, 36, 1024, "rank"),
    "direct_small_table_wide": (51, 1024, 756, "rank"),
    "direct_sixteen_waves": (300, 768, 4096, "rank"),
    "direct_sixteen_waves_same": (12, 192, 4001, "same"),
    "direct_sixteen_waves_odd": (1000, 33, 1500, "padded"),
    "counted_small_wide_table": (255, 2304, 1500, "rank"),
    "counted_above_the_direct_form": (3000, 64, 1025, "outside"),
    "direct_small_table_odd_width": (51, 333, 256, "padded"),
}


def tokens(kind, V, rows, seed):
    r = np.random.default_rng(seed)
    t = r.integers(0, V, rows)
    if kind == "rank":
        t = np.clip((float(V) ** r.random(rows)).astype(np.int64) - 1, 0, V - 1)
    if kind == "same":
        t[:] = V // 3
        t[::501] = V - 1
    if kind == "padded":
        t[r.random(rows) < 0.4] = -1
    if kind == "all_padding":
        t[:] = -1
    if kind == "outside":
        t[::3] = V
        t[1::7] = -2 ** 31
        t[2::11] = 2 ** 31 - 1
    return torch.from_numpy(t.astype(np.int32)).cuda()


@gpu
@pytest.mark.parametrize("name", list(EMBED))
def test_embedding_lookup_and_gradient(K, name):
    V, D, rows, kind = EMBED[name]
    g = rng(200)
    index = tokens(kind, V, rows, 1)
    there = (index >= 0) & (index < V)
    safe = torch.where(there, index, 0).long()
    scale = float(np.float32(D ** 0.5))
    table, out = randn(g, V, D), torch.full((rows, D), 7.0, device="cuda")
    K.embedding_fwd(table, index, out, scale=scale)
    assert torch.equal(out, torch.where(there[:, None], table[safe] * scale, 0.0))  # one product, rounded once
    dout = randn(g, rows, D)
    dout[~there] = float("nan")  # rows without a token add nothing, whatever they hold
    clean, there, safe = torch.where(there[:, None], dout, 0.0).double().cpu(), there.cpu(), safe.cpu()
    want = torch.zeros(V, D, dtype=torch.float64).index_add_(0, safe, clean) * scale
    mag = torch.zeros(V, D, dtype=torch.float64).index_add_(0, safe, clean.abs()) * scale
    count = torch.zeros(V, dtype=torch.float64).index_add_(0, safe, there.double())
    tol = (LAM * count.sqrt()[:, None] + 2) * U * mag
    dt = torch.full((V, D), float("nan"), device="cuda")
    K.embedding_bwd(dout, index, dt, scale=scale)
    within(dt, want, tol, "dtable")
    again = torch.full((V, D), float("nan"), device="cuda")
    K.embedding_bwd(dout, index, again, scale=scale)
    assert torch.equal(dt, again)
    base = randn(g, V, D)
    acc = base.clone()
    K.embedding_bwd(dout, index, acc, scale=scale, accumulate=True)
    total = base.double().cpu() + want
    within(acc, total, tol + 2 * U * total.abs(), "accumulated")
    untouched = count == 0
    assert torch.equal(acc.cpu()[untouched], base.cpu()[untouched])


@gpu
@pytest.mark.parametrize("V, D, rows, kind", [
    (2 ** 24 + 3, 1, 700001, "uniform"),     # four digits, every sort block with its largest share of tokens
    (2 ** 24 + 3, 1, 9000, "outside"),
    (100, 2, 1200007, "rank"),               # three levels of sums, runs over many chunks of each
    (3, 4, 2300000, "same"),
    (70000, 3, 1100000, "padded"),
    (255, 1, 1048577, "uniform"),            # one digit, and the padding's key behind it
    (256, 1, 1048576, "padded"),
])
def test_embedding_gradient_of_many_tokens(K, V, D, rows, kind):
    g = rng(204)
    index, dout = tokens(kind, V, rows, 7), randn(g, rows, D)
    there = (index >= 0) & (index < V)
    dout[~there] = float("nan")
    dt = torch.full((V, D), float("nan"), device="cuda")
    K.embedding_bwd(dout, index, dt, scale=0.5)
    there, safe = there.cpu(), torch.where(there, index, 0).long().cpu()
    clean = torch.where(there[:, None], dout.cpu(), 0.0).double()
    want = torch.zeros(V, D, dtype=torch.float64).index_add_(0, safe, clean) * 0.5
    mag = torch.zeros(V, D, dtype=torch.float64).index_add_(0, safe, clean.abs()) * 0.5
    count = torch.zeros(V, dtype=torch.float64).index_add_(0, safe, there.double())
    within(dt, want, (LAM * count.sqrt()[:, None] + 2) * U * mag, "dtable")
    again = torch.full((V, D), float("nan"), device="cuda")
    K.embedding_bwd(dout, index, again, scale=0.5)
    assert torch.equal(dt, again)


@gpu
@pytest.mark.parametrize("rows", [300, 5000, 20000])
def test_embedding_offsets_past_32_bits(K, rows):
    V, D = 2 ** 21 + 11, 1025
    index = torch.randint(V - 900, V, (rows,), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    index[::5] = torch.arange(len(index[::5]), dtype=torch.int32)
    table, index = torch.empty(V, D, device="cuda"), index.cuda()
    used = index.long().unique()
    table[used] = randn(rng(205), len(used), D)
    out = torch.empty(rows, D, device="cuda")
    K.embedding_fwd(table, index, out, scale=2.0)
    assert torch.equal(out, table[index.long()] * 2.0)
    dout = randn(rng(206), rows, D)
    K.embedding_bwd(dout, index, table, scale=0.5)  # into the same room
    want = torch.zeros(len(used), D, dtype=torch.float64, device="cuda")
    at = torch.searchsorted(used, index.long())
    want.index_add_(0, at, dout.double())
    mag = torch.zeros_like(want).index_add_(0, at, dout.double().abs())
    count = torch.bincount(at, minlength=len(used)).double()
    within(table[used], 0.5 * want, 0.5 * (LAM * count.sqrt()[:, None] + 2) * U * mag, "dtable")
    table[used] = 0
    assert not table.view(-1)[: 2 ** 31].any() and not table.view(-1)[2 ** 31:].any()


@gpu
def test_embedding_unaligned_and_empty(K):
    g = rng(201)
    V, D, rows = 50, 64, 200
    flat = randn(g, V * D + 1)[1:]
    table, index = flat.view(V, D), tokens("uniform", V, rows, 2)
    out = torch.empty(rows * D + 1, device="cuda")[1:].view(rows, D)
    K.embedding_fwd(table, index, out, scale=0.5)
    assert torch.equal(out, table[index.long()] * 0.5)
    dt = torch.empty(V * D + 1, device="cuda")[1:].view(V, D)
    K.embedding_bwd(out, index, dt, scale=1.0)
    want = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_add_(0, index.long(), out.double())
    within(dt, want, 64 * U * (1 + want.abs()), "dtable")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    dt.fill_(7.0)
    K.embedding_bwd(torch.empty(0, D, device="cuda"), none, dt)
    assert (dt == 0).all()
    K.embedding_fwd(table, none, torch.empty(0, D, device="cuda"))


@gpu
def test_embedding_lookup_of_more_rows_than_one_launch_takes(K):
    rows, V = 2 ** 29 + 5, 1000  # eight rows to a workgroup of 64 threads: 2^32 threads and a few
    table = randn(rng(203), V, 1)
    index = torch.arange(rows, dtype=torch.int32, device="cuda").remainder_(V)
    out = torch.full((rows, 1), 7.0, device="cuda")
    K.embedding_fwd(table, index, out, scale=0.5)
    whole = rows // V * V
    assert (out[:whole].view(-1, V) == 0.5 * table[:, 0]).all()
    assert torch.equal(out[whole:, 0], 0.5 * table[:rows - whole, 0])


@gpu
def test_embedding_gradient_captured_and_replayed(K):
    g = rng(202)
    V, D, rows = 3000, 96, 6000
    index, dout = tokens("rank", V, rows, 3), randn(g, rows, D)
    dt, eager = torch.empty(V, D, device="cuda"), torch.empty(V, D, device="cuda")
    ws = K.embedding_bwd(dout, index, dt)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.embedding_bwd(dout, index, dt, workspace=ws)
    for i in range(4):
        index.copy_(tokens(["rank", "padded", "same", "uniform"][i], V, rows, 10 + i))
        dout.copy_(randn(g, rows, D))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        K.embedding_bwd(dout, index, eager)
        assert torch.equal(dt, eager), i


# ------------------------------------------------------------------------- orthogonalised updates
COEF = (3.4445, -4.7750, 2.0315)


def newton_schulz(x, steps, coef, eps, dtype):
    a, b, c = (dtype(v) for v in coef)
    x = x.astype(np.float64)
    y = (x / (np.sqrt((x * x).sum()) + eps)).astype(dtype)
    tall = y.shape[0] > y.shape[1]
    y = y.T if tall else y
    for _ in range(steps):
        g = y @ y.T
        y = a * y + (b * g + c * (g @ g)) @ y
    return y.T if tall else y


def ns_tolerance(x, want, steps, coef, eps):
    """Frobenius bound.  The same steps in fp32 are off by some E.  Here the operands of the products carry
    22 instead of 24 bits: 4 u each, independent, so a sum of n terms gains 4 u / sqrt(n) of its norm
    product where the fp32 sum itself loses about u: the same order for n >= 16, and 4 E covers it.
    Short sums (n < 16): five steps of at most 12 u each, passed on with a factor of at most 4 in all."""
    plain = newton_schulz(x, steps, coef, eps, np.float32)
    return 4 * np.linalg.norm(plain - want) + 256 * U * np.linalg.norm(want)


ORTHO = {
    # rows, cols, batch, steps, pitch padding
    "one": (1, 1, 1, 5, 0),
    "row": (1, 70, 2, 5, 0),
    "column": (300, 1, 1, 5, 3),
    "square_96": (96, 96, 1, 5, 0),
    "square_64_batch": (64, 64, 5, 5, 0),
    "wide": (65, 200, 2, 5, 0),
    "tall": (257, 100, 2, 5, 1),
    "odd": (131, 129, 1, 3, 7),
    "no_steps": (40, 50, 2, 0, 2),
    "one_step": (50, 40, 1, 1, 0),
    "longer": (192, 576, 3, 5, 0),
    "ten_steps": (128, 128, 1, 10, 0),
    "one_launch_ragged": (33, 128, 3, 5, 0),
    "one_launch_tall": (127, 97, 2, 5, 3),
    "small_tiles": (257, 1000, 1, 5, 0),
    "small_tiles_thin": (3, 2500, 1, 5, 0),
    "tiles_64": (130, 520, 8, 5, 4),
    "tiles_64_tall": (700, 190, 9, 3, 1),
    "tiles_128": (300, 900, 9, 5, 0),
    "tiles_128_tall": (1001, 385, 7, 2, 0),
    "small_tiles_many": (200, 201, 11, 5, 0),
    "small_tiles_many_long": (777, 801, 1, 3, 0),
    "small_tiles_16": (513, 514, 1, 4, 2),
    "small_tiles_batch": (190, 192, 5, 5, 0),
    "thin_long": (100, 3300, 2, 5, 0),
    "thin_tall_padded": (3301, 70, 2, 3, 3),
    "small_tiles_tall_batch": (300, 130, 6, 5, 1),
}


@gpu
@pytest.mark.parametrize("name", list(ORTHO))
def test_newton_schulz(K, name):
    r, c, batch, steps, pad = ORTHO[name]
    g = rng(300 + list(ORTHO).index(name))
    full = randn(g, batch, r, c + pad) * 1e-3
    x = full[:, :, :c]
    out = torch.full((batch, r, c + pad), 7.0, device="cuda")
    K.newton_schulz(K.newton_schulz_args(x, out[:, :, :c], steps=steps, coefficients=COEF, eps=1e-7))
    assert (out[:, :, c:] == 7.0).all()
    for i in range(batch):
        h = x[i].cpu().numpy()
        want = newton_schulz(h, steps, COEF, 1e-7, np.float64)
        err = np.linalg.norm(out[i, :, :c].double().cpu().numpy() - want)
        assert err <= ns_tolerance(h, want, steps, COEF, 1e-7), (i, err, np.linalg.norm(want))
    # in place, the same bits
    inplace = full.clone()
    K.newton_schulz(K.newton_schulz_args(inplace[:, :, :c], inplace[:, :, :c], steps=steps, coefficients=COEF, eps=1e-7))
    assert torch.equal(inplace[:, :, :c], out[:, :, :c])


@gpu
@pytest.mark.parametrize("cus", [8, 64, 1024])
def test_newton_schulz_on_the_routes_of_other_devices(K, cus):
    K.planning_cu_count(cus)
    try:
        for i, (batch, r, c) in enumerate(((1, 257, 500), (3, 200, 300), (4, 130, 320), (2, 90, 700), (2, 300, 200))):
            x = randn(rng(900 + i), batch, r, c)
            out = torch.full_like(x, 7.0)
            K.newton_schulz(K.newton_schulz_args(x, out, steps=5, coefficients=COEF, eps=1e-7))
            for b in range(batch):
                want = newton_schulz(x[b].cpu().numpy(), 5, COEF, 1e-7, np.float64)
                err = np.linalg.norm(out[b].double().cpu().numpy() - want)
                assert err <= ns_tolerance(x[b].cpu().numpy(), want, 5, COEF, 1e-7), (batch, r, c, err)
    finally:
        K.planning_cu_count(0)


@gpu
def test_newton_schulz_orthogonalises(K):
    """With the convergent triple (15, -10, 3) / 8 the singular values go to 1."""
    x = randn(rng(320), 80, 120)
    out = torch.empty_like(x)
    K.newton_schulz(K.newton_schulz_args(x, out, steps=20, coefficients=(15 / 8, -10 / 8, 3 / 8), eps=0.0))
    s = torch.linalg.svdvals(out.double().cpu())
    assert (s - 1).abs().max() < 1e-4, (s.min(), s.max())


@gpu
def test_newton_schulz_scales(K):
    """Tiny, huge, zero and spiked matrices: the norm is formed in double precision."""
    g = rng(321)
    x = randn(g, 5, 70, 90)
    x[1] *= 1e-30
    x[2] *= 1e30
    x[3] = 0
    x[4] *= 1e-6
    x[4, 3, 5] = 1.0
    out = torch.empty_like(x)
    K.newton_schulz(K.newton_schulz_args(x, out, eps=0.0 + 1e-38))
    assert (out[3] == 0).all()
    for i in (0, 1, 2, 4):
        h = x[i].cpu().numpy()
        want = newton_schulz(h, 5, COEF, 1e-38, np.float64)
        # one strong direction beside a floor 1e-6 below: fp16 parts keep 2^-36 of the largest entry absolutely
        floor = 2.0 ** -36 * 3.4445 ** 5 * np.sqrt(h.size) if i == 4 else 0.0
        err = np.linalg.norm(out[i].double().cpu().numpy() - want)
        assert err <= ns_tolerance(h, want, 5, COEF, 1e-38) + floor, (i, err)


def graded(kind, level, batch, r, c, seed):
    """Matrices whose entries span many magnitudes: half of the rows `level` of the others, or one entry of 1 over a
    floor of `level`."""
    x = randn(rng(seed), batch, r, c)
    if kind == "cold rows":
        x[:, r // 2:] *= level
    else:
        x *= level
        x[:, r // 3, c // 4] = 1.0
    return x


def graded_tolerance(x, want, steps, rowwise):
    """Bound of each row's (column's) norm.  An operand is within 2 u of its value and the dropped product of two lo
    parts within 4 u, so a product is off by 8 u of its terms; a step rounds y (2 u), forms and rounds y y^T (8 + 2 u) and
    the polynomial (8 + 2 u), and multiplies (8 u): 30 u of a row, in five steps 150 u, passed on with a factor of at most
    4 relative to the row, which grows as its error does: 600 u.  The sums are those of the same steps in fp32, of
    which four times the error is taken.  Below 2^-25 a pair of y is within 2^-48: sqrt(n) of those a row, times 3.4445 a
    step and 1.41 for all of them."""
    axis = 1 if rowwise else 0
    plain = newton_schulz(x, steps, COEF, 1e-30, np.float32)
    norm = lambda z: np.linalg.norm(z, axis=axis)  # noqa: E731
    return 4 * norm(plain - want) + 600 * U * norm(want) + 1.41 * 3.4445 ** steps * np.sqrt(x.shape[axis]) * 2.0 ** -48


@gpu
@pytest.mark.parametrize("kind, level", [("cold rows", 1e-3), ("cold rows", 1e-6), ("cold rows", 1e-7), ("spike", 1e-6),
                                         ("spike", 1e-8)])
@pytest.mark.parametrize("cus, batch, r, c", [(0, 2, 70, 90), (0, 1, 128, 96), (0, 1, 200, 300), (0, 1, 513, 514),
                                              (10, 1, 200, 300), (4, 1, 200, 300), (4, 1, 300, 200)],
                         ids=["one", "one_tall", "small", "lower", "64", "128", "128_tall"])
def test_newton_schulz_keeps_small_entries(K, kind, level, cus, batch, r, c):
    """Each row is as close as its own size allows, however large the others are.  (cus: tiles of 64 and 128 at these
    sizes, as a device with so few CUs would take them.)"""
    K.planning_cu_count(cus)
    try:
        x = graded(kind, level, batch, r, c, 350)
        out = torch.empty_like(x)
        K.newton_schulz(K.newton_schulz_args(x, out, steps=5, coefficients=COEF, eps=1e-30))
        for b in range(batch):
            h = x[b].cpu().numpy()
            want = newton_schulz(h, 5, COEF, 1e-30, np.float64)
            err = np.linalg.norm(out[b].double().cpu().numpy() - want, axis=1)
            over = err / graded_tolerance(h, want, 5, True)
            assert (over <= 1).all(), (b, int(over.argmax()), over.max(), (err / np.linalg.norm(want, axis=1)).max())
    finally:
        K.planning_cu_count(0)


@gpu
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shape", [(96, 288, 3), (288, 96, 2), (10, 192, 1)])
def test_muon_steps(K, nesterov, shape):
    r, c, batch = shape
    g = rng(330)
    p, m = randn(g, batch, r, c) * 0.02, torch.zeros(batch, r, c, device="cuda")
    p64, m64 = p.double().cpu().numpy(), m.double().cpu().numpy()
    lr, mu, wd, us, gs = 0.02, 0.95, 0.1, 1.5, 0.25
    for step in range(3):
        grad = randn(g, batch, r, c) * 1e-2
        K.muon(K.muon_args(p, grad, m, lr=lr, momentum=mu, weight_decay=wd, update_scale=us, grad_scale=gs,
                           nesterov=nesterov))
        gd = grad.double().cpu().numpy() * gs
        m64 = mu * m64 + gd
        tol_m = (step + 1) * 4 * U * (np.abs(m64) + np.abs(gd) + 1e-2)
        assert (np.abs(m.double().cpu().numpy() - m64) <= tol_m).all()
        u = gd + mu * m64 if nesterov else m64
        for i in range(batch):
            o = newton_schulz(u[i].astype(np.float32), 5, COEF, 1e-7, np.float64)
            p64[i] = p64[i] * (1 - lr * wd) - lr * us * o
            # the direction: bound of the products plus what 12 u in u becomes (a factor of at most 3.4445^5)
            e = ns_tolerance(u[i].astype(np.float32), o, 5, COEF, 1e-7) + 12 * U * 485
            err = np.linalg.norm(p[i].double().cpu().numpy() - p64[i])
            assert err <= (step + 1) * (lr * us * e + 4 * U * np.linalg.norm(p64[i])), (step, i, err)


MUON = {
    # CUs to plan for, batch, rows, cols, floats between rows, between matrices, in front
    "one": (0, 3, 33, 128, 0, 0, 0),
    "one_tall": (0, 2, 128, 97, 0, 0, 0),
    "one_odd": (0, 2, 70, 90, 0, 0, 0),
    "one_padded": (0, 2, 64, 96, 4, 8, 4),
    "one_padded_odd": (0, 2, 96, 64, 3, 5, 1),
    "one_row": (0, 2, 1, 100, 0, 0, 1),
    "small": (0, 2, 150, 200, 0, 0, 0),
    "small_padded": (0, 2, 150, 200, 4, 4, 0),
    "small_unaligned": (0, 1, 200, 131, 0, 0, 1),
    "small_tall_padded_odd": (0, 2, 300, 130, 1, 2, 3),
    "64": (10, 1, 200, 300, 0, 0, 0),
    "64_tall": (10, 1, 300, 200, 0, 0, 0),
    "64_padded": (20, 2, 190, 300, 4, 12, 4),
    "64_tall_odd": (20, 2, 301, 190, 2, 1, 1),
    "128": (4, 1, 200, 300, 0, 0, 0),
    "128_tall": (4, 1, 300, 200, 0, 0, 0),
    "128_padded": (8, 2, 200, 300, 4, 0, 0),
    "128_odd": (8, 2, 129, 259, 0, 0, 1),
    "128_tall_odd": (8, 2, 259, 130, 3, 7, 2),
}


@gpu
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("name", list(MUON))
def test_muon_in_every_form_and_layout(K, name, nesterov):
    """p and m of three steps, and nothing else of their buffers: what lies between rows and matrices stays as it was."""
    cus, batch, r, c, pad, gap, front = MUON[name]
    ld, g = c + pad, rng(370 + list(MUON).index(name))
    stride = r * ld + gap
    size = front + batch * stride

    def matrices(flat):
        return flat.as_strided((batch, r, c), (stride, ld, 1), front)

    buffers = [randn(g, size) * s for s in (0.02, 1e-2, 3e-3)]
    p, grad, m = (matrices(b) for b in buffers)
    p64, m64 = p.double().cpu().numpy(), m.double().cpu().numpy()
    lr, mu, wd, us, gs = 0.02, 0.9, 0.2, 1.5, 0.25
    outside = torch.ones(size, dtype=torch.bool, device="cuda")
    matrices(outside)[:] = False
    kept = [b[outside].clone() for b in buffers]
    K.planning_cu_count(cus)
    try:
        args = K.muon_args(p, grad, m, lr=lr, momentum=mu, weight_decay=wd, update_scale=us, grad_scale=gs, nesterov=nesterov)
        for step in range(3):
            grad.copy_(randn(g, batch, r, c) * 1e-2)
            before = grad.clone()
            K.muon(args)
            assert torch.equal(grad, before)
            gd = grad.double().cpu().numpy() * gs
            m64 = mu * m64 + gd
            # three roundings of at most u of each term, a step
            tol_m = (step + 1) * 4 * U * (np.abs(m64) + np.abs(gd) + 1e-2)
            assert (np.abs(m.double().cpu().numpy() - m64) <= tol_m).all(), step
            u = gd + mu * m64 if nesterov else m64
            for i in range(batch):
                o = newton_schulz(u[i].astype(np.float32), 5, COEF, 1e-7, np.float64)
                p64[i] = p64[i] * (1 - lr * wd) - lr * us * o
                # the direction: bound of the products plus what 12 u in u becomes (a factor of at most 3.4445^5)
                e = ns_tolerance(u[i].astype(np.float32), o, 5, COEF, 1e-7) + 12 * U * 485
                err = np.linalg.norm(p[i].double().cpu().numpy() - p64[i])
                assert err <= (step + 1) * (lr * us * e + 4 * U * np.linalg.norm(p64[i])), (step, i, err)
    finally:
        K.planning_cu_count(0)
    for b, k in zip(buffers, kept):
        assert torch.equal(b[outside], k)


@gpu
@pytest.mark.parametrize("r, c", [(60, 100), (140, 100), (300, 500)])
def test_muon_offsets_past_32_bits(K, r, c):
    """Rows and matrices far apart: the second matrix starts more than 2^31 elements behind the first."""
    ld, stride, g = 2 ** 20, 2 ** 31 + 64, rng(395)
    room = torch.empty(stride + r * ld, device="cuda")
    p, grad, m = (room.as_strided((2, r, c), (stride, ld, 1), i * 1024).copy_(randn(g, 2, r, c) * x)
                  for i, x in enumerate((0.02, 1e-2, 3e-3)))
    near = [t.contiguous() for t in (p, grad, m)]
    for t in ((p, grad, m), near):
        K.muon(K.muon_args(*t, lr=0.1, weight_decay=0.1))
    assert torch.equal(m, near[2])
    # a row pitch may choose other loads, not other sums
    assert (p - near[0]).abs().max() <= 4 * U
    out = torch.empty_like(near[1])
    K.newton_schulz(K.newton_schulz_args(near[1], out))
    K.newton_schulz(K.newton_schulz_args(grad, p))
    assert torch.equal(p, out)


@gpu
def test_muon_captured_and_replayed(K):
    g = rng(340)
    shape = (2, 64, 160)
    p, m = randn(g, *shape), torch.zeros(*shape, device="cuda")
    grad = torch.empty(*shape, device="cuda")
    pe, me = p.clone(), m.clone()
    a, e = K.muon_args(p, grad, m, lr=0.1), K.muon_args(pe, grad, me, lr=0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.muon(a)
    for i in range(4):
        grad.copy_(randn(g, *shape))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        K.muon(e)
        assert torch.equal(p, pe) and torch.equal(m, me), i


# ------------------------------------------------------------------------------------- refusals
def _xargs(vitk, **kw):
    a = vitk.CrossSdpaArgs()
    d = dict(B=2, H=4, Hkv=2, Nq=3, Nk=5, dh=8, scale=1.0, q=4096, ld_q=32, k=8192, ld_k=16, v=12288, ld_v=16, out=16384,
             ld_out=32, stats=20480, dout=24576, ld_dout=32, dq=28672, ld_dq=32, dk=32768, ld_dk=16, dv=36864, ld_dv=16,
             workspace=40960, workspace_bytes=1 << 20)
    d.update(kw)
    for n, x in d.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("change, message", [
    (dict(B=-1), "negative size"), (dict(Hkv=3), "query heads over"), (dict(Hkv=0), "query heads over"),
    (dict(H=0), "query heads over"), (dict(dh=0), "outside"), (dict(dh=129), "outside"),
    (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(q=0), "null pointer"),
    (dict(k=0), "null pointer"), (dict(out=0), "null pointer"), (dict(ld_q=31), "pitch"), (dict(ld_k=15), "pitch"),
    (dict(ld_out=1), "pitch"), (dict(out=4096), "one of the inputs"), (dict(reserved=1), "reserved"), (dict(Nq=2 ** 30, H=8), "too many rows")])
def test_cross_attention_refuses(change, message):
    from visiontransformer_amd import vitk
    d = vitk.dll()
    for fn in (d.vitk_cross_sdpa_fwd, d.vitk_cross_sdpa_bwd):
        assert fn(C.byref(_xargs(vitk, **change)), None) != 0
        assert message in d.vitk_last_error().decode()


@pytest.mark.parametrize("change", [dict(Nq=2 ** 30, H=8), dict(Nq=2 ** 31 - 1, H=2), dict(Nk=2 ** 31 - 1)])
def test_cross_attention_needs_no_workspace_for_what_it_refuses(change):
    from visiontransformer_amd import vitk
    d = vitk.dll()
    a = _xargs(vitk, **change)
    assert d.vitk_cross_sdpa_fwd_workspace_bytes(C.byref(a)) == 0 and d.vitk_cross_sdpa_bwd_workspace_bytes(C.byref(a)) == 0


@pytest.mark.parametrize("change, forward, backward", [
    (dict(B=2 ** 21, H=8, Hkv=8, Nq=1, Nk=5), True, True),  # 2^24 workgroups of four waves
    (dict(B=2 ** 20, H=15, Hkv=15, Nq=1, Nk=5), False, False),
    (dict(B=2 ** 20, H=8, Hkv=8, Nq=40, Nk=70), False, True),  # 2^23 of eight waves
    (dict(B=2 ** 21, H=8, Hkv=8, Nq=40, Nk=70), True, True),
    (dict(B=1, H=1, Hkv=1, Nq=2 ** 30, Nk=5), True, False)])  # 2^24 blocks of 64 rows
def test_cross_attention_refuses_more_threads_than_a_launch_has(change, forward, backward):
    """Before anything is launched (what is not refused fails here only for want of a device)."""
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    from visiontransformer_amd import vitk
    d = vitk.dll()
    a = _xargs(vitk, dh=1, workspace_bytes=1 << 62, **{"ld_" + n: 16 for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv")},
               **change)
    for fn, refused in ((d.vitk_cross_sdpa_fwd, forward), (d.vitk_cross_sdpa_bwd, backward)):
        assert fn(C.byref(a), None) != 0
        assert ("too many rows" in d.vitk_last_error().decode()) == refused, d.vitk_last_error()


@pytest.mark.parametrize("batch, cols, refused", [(2 ** 22, 16, True), (2 ** 22 - 1, 16, False), (2 ** 18, 130, True),
                                                  (2 ** 18 - 1, 130, False)])
def test_newton_schulz_refuses_more_threads_than_a_launch_has(batch, cols, refused):
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    from visiontransformer_amd import vitk
    d = vitk.dll()
    change = dict(batch=batch, rows=16, cols=cols, steps=1, workspace_bytes=1 << 62)
    for fn, a in ((d.vitk_newton_schulz_f32, _nargs(vitk, vitk.NewtonSchulzArgs, **change)),
                  (d.vitk_muon_f32, _nargs(vitk, vitk.MuonArgs, **change))):
        assert fn(C.byref(a), None) != 0
        assert ("too many matrices" in d.vitk_last_error().decode()) == refused, d.vitk_last_error()


@pytest.mark.parametrize("change, message", [
    (dict(dout=0), "null pointer"), (dict(dq=0), "null pointer"), (dict(dk=0), "null pointer"), (dict(dv=0), "null pointer"),
    (dict(stats=0), "null pointer"), (dict(dq=24576), "one of the inputs"), (dict(dk=8192), "one of the inputs"),
    (dict(dv=16384), "one of the inputs"), (dict(dv=32768), "share"), (dict(dq=36864), "share"), (dict(ld_dq=31), "pitch"), (dict(ld_dv=15), "pitch"),
    (dict(Nk=70, workspace=0), "workspace"), (dict(Nk=70, workspace_bytes=4), "workspace"),
    (dict(Nk=70, workspace=40964), "aligned"), (dict(Nq=1000, workspace=0), "workspace")])
def test_cross_attention_backward_refuses(change, message):
    from visiontransformer_amd import vitk
    d = vitk.dll()
    assert d.vitk_cross_sdpa_bwd(C.byref(_xargs(vitk, **change)), None) != 0
    assert message in d.vitk_last_error().decode()


def test_cross_attention_refuses_null_arguments_and_a_missing_workspace():
    from visiontransformer_amd import vitk
    d = vitk.dll()
    assert d.vitk_cross_sdpa_fwd(None, None) != 0
    assert d.vitk_cross_sdpa_bwd(None, None) != 0
    a = _xargs(vitk, B=1, H=1, Hkv=1, Nq=1, Nk=100000, dh=64, ld_q=64, ld_k=64, ld_v=64, ld_out=64, workspace=0)
    assert d.vitk_cross_sdpa_fwd_workspace_bytes(C.byref(a)) > 0  # split over keys
    assert d.vitk_cross_sdpa_fwd(C.byref(a), None) != 0
    assert "workspace" in d.vitk_last_error().decode()


@pytest.mark.parametrize("name, args, message", [
    ("vitk_embedding_fwd", (4096, 10, 4096, -1, 8, 1.0, 8192, None), "bad shape"),
    ("vitk_embedding_fwd", (4096, 10, 8192, 3, 8, 1.0, 4096, None), "is the table"),
    ("vitk_embedding_bwd", (4096, 8192, 3, 10, 8, 1.0, 0, 4096, 12288, 1 << 20, None), "is dout"),
    ("vitk_embedding_fwd", (None, 10, 4096, 3, 8, 1.0, 4096, None), "null pointer"),
    ("vitk_embedding_fwd", (4096, 10, None, 3, 8, 1.0, 4096, None), "null pointer"),
    ("vitk_embedding_fwd", (4096, 2 ** 31, 4096, 3, 8, 1.0, 8192, None), "table of"),
    ("vitk_embedding_bwd", (4096, 4096, 3, -10, 8, 1.0, 0, 4096, 4096, 1 << 20, None), "bad shape"),
    ("vitk_embedding_bwd", (None, 4096, 3, 10, 8, 1.0, 0, 4096, 4096, 1 << 20, None), "null pointer"),
    ("vitk_embedding_bwd", (4096, 4096, 3, 10, 8, 1.0, 0, None, 4096, 1 << 20, None), "null pointer"),
    ("vitk_embedding_bwd", (4096, 4096, 3, 50000, 8, 1.0, 0, 8192, None, 1 << 20, None), "workspace"),
    ("vitk_embedding_bwd", (4096, 4096, 20000, 10, 8, 1.0, 0, 8192, 4096, 16, None), "workspace"),
    ("vitk_embedding_bwd", (4096, 4096, 20000, 10, 8, 1.0, 0, 8192, 4100, 1 << 20, None), "aligned"),
    ("vitk_embedding_bwd", (4096, 4096, 2 ** 31, 10, 8, 1.0, 0, 8192, 4096, 1 << 20, None), "tokens over"),
])
def test_embedding_refuses(name, args, message):
    from visiontransformer_amd import vitk
    with pytest.raises(vitk.VitkError, match=message):
        vitk.call(name, *args)


def _nargs(vitk, cls, **kw):
    a = cls()
    d = dict(rows=200, cols=200, batch=2, steps=5, a=COEF[0], b=COEF[1], c=COEF[2], eps=1e-7, workspace=4096, workspace_bytes=1 << 30)
    if cls is vitk.MuonArgs:
        d.update(p=4096, g=8192, m=16384, ld=200, stride=40000)
    else:
        d.update(x=4096, out=4096, ld_x=200, ld_out=200, stride_x=40000, stride_out=40000)
    d.update(kw)
    for n, x in d.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("change, message", [
    (dict(rows=-1), "bad shape"), (dict(cols=2 ** 21), "bad shape"), (dict(steps=-1), "steps"), (dict(steps=33), "steps"),
    (dict(a=9.0), "bounded"), (dict(c=float("nan")), "bounded"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(workspace=0), "workspace"), (dict(workspace_bytes=64), "workspace"), (dict(workspace=4104), "aligned")])
def test_newton_schulz_and_muon_refuse(change, message):
    from visiontransformer_amd import vitk
    d = vitk.dll()
    for fn, cls in ((d.vitk_newton_schulz_f32, vitk.NewtonSchulzArgs), (d.vitk_muon_f32, vitk.MuonArgs)):
        assert fn(C.byref(_nargs(vitk, cls, **change)), None) != 0
        assert message in d.vitk_last_error().decode()


@pytest.mark.parametrize("cls, change, message", [
    ("NewtonSchulzArgs", dict(x=0), "null pointer"), ("NewtonSchulzArgs", dict(out=0), "null pointer"),
    ("NewtonSchulzArgs", dict(ld_x=7), "pitch"), ("NewtonSchulzArgs", dict(ld_x=201, stride_x=40200), "one layout"),
    ("NewtonSchulzArgs", dict(stride_x=0), "one layout"), ("NewtonSchulzArgs", dict(stride_out=63), "overlap"),
    ("MuonArgs", dict(p=0), "null pointer"), ("MuonArgs", dict(m=8192), "different buffers"),
    ("MuonArgs", dict(ld=7), "pitch"), ("MuonArgs", dict(stride=63), "overlap")])
def test_newton_schulz_and_muon_refuse_their_own(cls, change, message):
    from visiontransformer_amd import vitk
    d = vitk.dll()
    fn = d.vitk_muon_f32 if cls == "MuonArgs" else d.vitk_newton_schulz_f32
    assert fn(C.byref(_nargs(vitk, getattr(vitk, cls), **change)), None) != 0
    assert message in d.vitk_last_error().decode()


def test_bindings_refuse_wrong_tensors():
    from visiontransformer_amd import vitk
    cpu = torch.zeros(2, 3, 4, 8)
    with pytest.raises(vitk.VitkError, match="CUDA"):
        vitk.cross_sdpa_args(cpu, cpu, cpu, cpu)
    with pytest.raises(vitk.VitkError, match="CUDA"):
        vitk.embedding_fwd(torch.zeros(4, 4), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4))
    with pytest.raises(vitk.VitkError, match="CUDA"):
        vitk.newton_schulz_args(torch.zeros(4, 4), torch.zeros(4, 4))
    with pytest.raises(vitk.VitkError, match="CUDA"):
        vitk.muon_args(torch.zeros(4, 4), torch.zeros(4, 4), torch.zeros(4, 4), lr=0.1)


def test_a_workspace_with_gaps_or_repeated_elements_is_refused():
    from visiontransformer_amd import vitk

    class OnTheDevice:  # a tensor's strides where there is no device
        is_cuda = True

        def __init__(self, t):
            self.is_contiguous, self.nbytes, self.data_ptr = t.is_contiguous, t.nbytes, t.data_ptr

    whole = torch.empty(64)
    assert vitk._room(OnTheDevice(whole)) == (whole.data_ptr(), 256)
    for t in (whole[:1].expand(1 << 20), whole[::2], whole.view(8, 8).t()):
        with pytest.raises(vitk.VitkError, match="contiguous"):
            vitk._room(OnTheDevice(t))
    with pytest.raises(vitk.VitkError, match="CUDA"):
        vitk._room(whole)


@gpu
def test_the_bindings_refuse_a_repeated_workspace(K):
    g = rng(6)
    one = torch.zeros(1, device="cuda").expand(1 << 24)
    q, k = randn(g, 1, 1, 1, 64), randn(g, 1, 20000, 1, 64)
    with pytest.raises(K.VitkError, match="contiguous"):
        K.cross_sdpa_args(q, k, k, torch.empty_like(q), workspace=one)
    w = randn(g, 200, 200)
    with pytest.raises(K.VitkError, match="contiguous"):
        K.newton_schulz_args(w, torch.empty_like(w), workspace=one)
    with pytest.raises(K.VitkError, match="contiguous"):
        K.muon_args(w, randn(g, 200, 200), randn(g, 200, 200), lr=0.1, workspace=one)
    index = torch.zeros(20000, dtype=torch.int32, device="cuda")
    with pytest.raises(K.VitkError, match="contiguous"):
        K.embedding_bwd(randn(g, 20000, 4), index, torch.empty(3000, 4, device="cuda"), workspace=one)


@gpu
def test_the_bindings_refuse_another_device(K):
    g = rng(5)
    x, out = randn(g, 16, 16), torch.empty(16, 16, device="cuda")
    args = K.newton_schulz_args(x, out)
    assert args.device == torch.cuda.current_device()
    args.device += 1  # as if its tensors were there
    with pytest.raises(K.VitkError, match="current one"):
        K.newton_schulz(args)
    with pytest.raises(K.VitkError, match="current one"):
        K.stream(torch.cuda.current_device() + 1)
    with pytest.raises(K.VitkError, match="different devices"):
        K._one_device(x, torch.empty(2))


def test_newton_schulz_takes_every_triple_that_stays_and_no_other():
    """A coarse search over triples: what is accepted stays within the bounds on a fine grid."""
    from visiontransformer_amd import vitk
    d = vitk.dll()
    r = np.random.default_rng(9)
    t0 = np.linspace(0.0, 1.0, 20001)
    seen = set()
    for _ in range(400):
        a, b, c = (np.float32(x) for x in r.uniform((0.0, -12.0, -2.0), (6.0, 6.0, 8.0)))
        if r.random() < 0.2:
            c = np.float32(0.0)
        if r.random() < 0.1:
            b = np.float32(0.0)
        steps = int(r.integers(1, 9))
        args = _nargs(vitk, vitk.NewtonSchulzArgs, a=a, b=b, c=c, steps=steps, workspace=0)  # refused either way
        assert d.vitk_newton_schulz_f32(C.byref(args), None) != 0
        taken = "bounded" not in d.vitk_last_error().decode()
        seen.add(taken)
        if taken:
            t = t0.copy()
            for _ in range(steps):
                poly = float(b) * t ** 2 + float(c) * t ** 4
                assert (np.abs(poly) < 31.0).all()
                t = float(a) * t + poly * t
                assert (np.abs(t) <= 4.0 + 1e-9).all(), (a, b, c, steps)
    assert seen == {True, False}


def taken(a, b, c, steps):
    """Are these coefficients accepted?  (The call is refused either way, for its workspace.)"""
    from visiontransformer_amd import vitk
    d = vitk.dll()
    args = _nargs(vitk, vitk.NewtonSchulzArgs, a=a, b=b, c=c, steps=steps, workspace=0)
    assert d.vitk_newton_schulz_f32(C.byref(args), None) != 0
    message = d.vitk_last_error().decode()
    assert "bounded" in message or "workspace" in message
    return "bounded" not in message


@pytest.mark.parametrize("c", [0.0] + [sign * 10.0 ** e for e in (-30, -20, -16, -15, -13, -12, -9, -6) for sign in (1, -1)])
@pytest.mark.parametrize("a, b", [(15.0, -14.0), (8.0, -7.5), (-15.0, 14.0), (2.0, -1.0), (1.5, -0.5), (-1.5, 0.5), (0.5, 0.25)])
def test_newton_schulz_coefficients_next_to_a_cubic(a, b, c):
    """A fifth-order term that is too small to matter changes nothing: the extremum is that of a t + b t^3."""
    t, stays = np.linspace(0.0, 1.0, 20001), True
    for _ in range(5):
        poly = b * t ** 2 + c * t ** 4
        t = a * t + poly * t
        stays = stays and bool((np.abs(poly) < 31.0).all() and (np.abs(t) <= 4.0).all())
        if not stays:
            break
    assert taken(a, b, c, 5) == stays


KEEPING = [COEF, (15 / 8, -10 / 8, 3 / 8), (1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (3.0, -3.0, 1.0)]


@pytest.mark.parametrize("a, b, c", [(5.0, -20.0, 16.0), (3.0, -4.0, 0.0), (3.0, -2.0, 0.0), (-5.0, 20.0, -16.0)])
def test_newton_schulz_refuses_coefficients_that_rounding_carries_out_of_range(a, b, c):
    """Exactly, each of these keeps [0, 1] (or what it makes of it) for ever; beside the end it grows by 9 to 25 a step."""
    assert taken(a, b, c, 1)
    assert not taken(a, b, c, 12)


@pytest.mark.parametrize("coef", KEEPING)
def test_newton_schulz_takes_convergent_coefficients_for_every_number_of_steps(coef):
    assert all(taken(*coef, steps) for steps in range(33))


@gpu
@pytest.mark.parametrize("coef", KEEPING)
@pytest.mark.parametrize("shape", [(96, 120), (150, 200)])
def test_newton_schulz_of_one_direction_stays_in_range(K, shape, coef):
    """The one singular value starts at 1 but for its rounding; in each of 32 steps it stays below 4."""
    x = randn(rng(360), shape[0], 1) * randn(rng(361), 1, shape[1])
    out = torch.empty_like(x)
    K.newton_schulz(K.newton_schulz_args(x, out, steps=32, coefficients=coef, eps=0.0))
    assert torch.isfinite(out).all() and torch.linalg.norm(out.double().cpu()) <= 4.0 * min(shape) ** 0.5


# ---------------------------------------------------------------------------- the run together
@gpu
def test_all_of_them_captured_in_one_graph(K):
    """Few keys (one kernel in the backward), tokens placed by counting, one launch of Newton-Schulz."""
    g = rng(77)
    x, out = randn(g, 96, 96), torch.empty(96, 96, device="cuda")
    q, k, v, dout = randn(g, 2, 70, 4, 64), randn(g, 2, 40, 4, 64), randn(g, 2, 40, 4, 64), randn(g, 2, 70, 4, 64)
    o, dq, dk, dv = (torch.empty_like(t) for t in (q, q, k, v))
    ns = K.newton_schulz_args(x, out)
    attn = K.cross_sdpa_args(q, k, v, o, stats=torch.empty(8, 70, 2, device="cuda"), dout=dout, dq=dq, dk=dk, dv=dv)
    index = tokens("rank", 20000, 3000, 4)
    d, dtable = randn(g, 3000, 64), torch.empty(20000, 64, device="cuda")
    workspace = torch.empty(K.dll().vitk_embedding_bwd_workspace_bytes(3000, 20000, 64) // 4 + 1, device="cuda")

    def run():
        K.newton_schulz(ns)
        K.cross_sdpa_fwd(attn)
        K.cross_sdpa_bwd(attn)
        K.embedding_bwd(d, index, dtable, workspace=workspace)

    results = (out, o, dq, dk, dv, dtable)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(3):
        for t in (x, q, k, v, dout, d):
            t.mul_(1.25)
        for t in results:
            t.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in results]
        run()
        for a, b in zip(replayed, results):
            assert torch.equal(a, b), i


@gpu
def test_the_bindings_follow_the_current_stream(K):
    assert K.stream() == torch.cuda.current_stream().cuda_stream
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        assert K.stream() == torch.cuda.current_stream().cuda_stream != 0
    assert K.stream() == torch.cuda.current_stream().cuda_stream


@gpu
def test_decoder_step_on_the_encoders_states(K):
    """One training step of a small decoder on a ViT encoder, every piece by the library: token embeddings, query
    projection, cross attention to the encoder's final states (ragged: one image has none), output
    projection to a vocabulary, softmax cross-entropy, the way back, the gradient of the embedding
    table and a Muon step on the two projections -- against float64 autograd on the CPU."""
    import vitlibs as V
    from visiontransformer_amd import host
    host.init(0)
    host.use_torch_stream()
    cfgd = V.TINY
    model = host.Model(host.Config.make(**cfgd))
    model.set_params(V.init_params(V.Cfg.make(**cfgd), 3))
    B, T, vocab, D, H = 4, 7, 50, cfgd["embedding_dim"], cfgd["num_heads"]
    dh, g = D // H, rng(400)
    acts, _ = model.forward_trace(torch.from_numpy(V.rng_normal(4, B, cfgd["in_channels"], cfgd["image_size"],
                                                                cfgd["image_size"])).cuda())
    states = acts[-1].contiguous()  # [B, N, D] behind the final norm
    N = states.shape[1]
    klen = torch.tensor([N, 0, N - 1, 2], dtype=torch.int32, device="cuda")
    index = torch.randint(0, vocab, (B * T,), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    index[5:7] = -1  # padding
    target = torch.randint(0, vocab, (B * T,), generator=torch.Generator().manual_seed(2))
    onehot = torch.nn.functional.one_hot(target, vocab).float().cuda()
    index = index.cuda()
    table, wq, wk, wv, wo = (randn(g, *s) * 0.3 for s in ((vocab, D), (D, D), (D, D), (D, D), (D, vocab)))
    rows, keys = B * T, B * N
    e = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
    emb, q, k, v, ctx, logits = e(rows, D), e(rows, D), e(keys, D), e(keys, D), e(rows, D), e(rows, vocab)
    scale = D ** 0.5
    K.embedding_fwd(table, index, emb, scale=scale)
    K.gemm(emb, wq, q, rows, D, D)
    K.gemm(states, wk, k, keys, D, D)
    K.gemm(states, wv, v, keys, D, D)
    dctx, dq, dk, dv = e(rows, D), e(rows, D), e(keys, D), e(keys, D)
    shape = lambda t, n: t.view(B, n, H, dh)  # noqa: E731
    args = K.cross_sdpa_args(shape(q, T), shape(k, N), shape(v, N), shape(ctx, T), key_len=klen, stats=e(B * H, T, 2),
                             dout=shape(dctx, T), dq=shape(dq, T), dk=shape(dk, N), dv=shape(dv, N))
    K.cross_sdpa_fwd(args)
    K.gemm(ctx, wo, logits, rows, vocab, D)
    dlogits, probs, out2, ws = e(rows, vocab), e(rows, vocab), e(2), e(2 * rows)
    K.call("vitk_softmax_ce", logits, onehot, rows, vocab, None, float(rows), dlogits, probs, out2, ws, ws.numel() * 4,
           K.stream())
    dwo, dwq, demb, dtable = e(D, vocab), e(D, D), e(rows, D), e(vocab, D)
    K.gemm(ctx, dlogits, dwo, D, vocab, rows, trans_a=True)
    K.gemm(dlogits, wo, dctx, rows, D, vocab, trans_b=True)
    K.cross_sdpa_bwd(args)
    K.gemm(emb, dq, dwq, D, D, rows, trans_a=True)
    K.gemm(dq, wq, demb, rows, D, D, trans_b=True)
    K.embedding_bwd(demb, index, dtable, scale=scale)
    # the same in float64
    leaf = {n: t.double().cpu().requires_grad_() for n, t in (("table", table), ("wq", wq), ("wo", wo), ("k", k), ("v", v))}
    idx = index.long().cpu()
    there = (idx >= 0)[:, None]
    emb64 = torch.where(there, leaf["table"][idx.clamp(min=0)] * scale, 0.0)
    q64 = (emb64 @ leaf["wq"]).view(B, T, H, dh)
    k64, v64 = (leaf[n].view(B, N, H, dh) for n in ("k", "v"))
    out = []
    for b in range(B):
        n = int(klen[b])
        if n == 0:
            out.append(torch.zeros(T, D, dtype=torch.float64))
            continue
        s = torch.einsum("qhd,khd->hqk", q64[b], k64[b, :n]) * dh ** -0.5
        out.append(torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v64[b, :n]).reshape(T, D))
    ctx64 = torch.cat(out)
    loss = torch.nn.functional.cross_entropy(ctx64 @ leaf["wo"], target)
    loss.backward()
    assert abs(out2[0].item() - loss.item()) <= 1e-5 * abs(loss.item())
    # sums of at most B T vocab = 1400 terms in fp32, five products deep: LAM sqrt(1400) u = 1.3e-5 of the largest entry each
    for name, got in (("wo", dwo), ("wq", dwq), ("table", dtable), ("k", dk), ("v", dv)):
        want = leaf[name].grad.reshape(got.shape)
        assert (got.double().cpu() - want).abs().max() <= 5 * 1.3e-5 * want.abs().max(), name
    # and the step on both projections
    for p, grad in ((wq, dwq), (wo, dwo)):
        before, m = p.double().cpu(), torch.zeros_like(p)
        K.muon(K.muon_args(p, grad, m, lr=0.05, momentum=0.9, nesterov=False))
        h = grad.cpu().numpy()
        o = newton_schulz(h, 5, COEF, 1e-7, np.float64)
        err = np.linalg.norm(p.double().cpu().numpy() - (before.numpy() - 0.05 * o))
        assert err <= 0.05 * ns_tolerance(h, o, 5, COEF, 1e-7) + 4 * U * np.linalg.norm(before.numpy())
    model.close()
