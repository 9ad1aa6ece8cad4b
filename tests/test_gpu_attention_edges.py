"""The attention operators where they went wrong or could: unknown sequences among known ones, pages that a row does
not see, values that are not finite, scratch and captured graphs, refused calls. Plain forms and the derivation of the
tolerances are those of test_gpu_attention.py."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_attention import (M, PAGE, U, check_rows, cu_of, filled_cache, held_rows, i32,  # noqa: E402,F401
                                plain_attention)

pytestmark = pytest.mark.gpu


def check_known(codes, scales, tables, lens, seqs, rows, q, out, lse, window=0, sinks=0, vmax_of=None):
    """attend's rows of every listed sequence against the plain form; unknown sequences, and rows beyond a
    sequence's length, are empty."""
    d = q.shape[2]
    qn, on, ln = q.double().cpu().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy()
    at = 0
    for s, m in zip(seqs, rows):
        known = 0 <= s < len(lens)
        n = lens[s] if known else 0
        none = max(0, m - n)
        assert np.all(on[at:at + none] == 0) and np.all(ln[at:at + none] == -np.inf)
        if known and m > none:
            k, present = held_rows(codes, scales, tables[s], n, 0)
            v, _ = held_rows(codes, scales, tables[s], n, 1)
            lo, hi = at + none, at + m
            want, wl, big = plain_attention(qn[lo:hi], k, v, n - (m - none), True, window, sinks, d ** -0.5, present)
            check_rows(on[lo:hi], ln[lo:hi], want, wl, big, d, n, np.abs(v).max(), U[q.dtype], 2.0 ** -11)
        at += m


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_unknown_sequences_between_known_ones(M, dev, d, dtype):
    """More sequences than the kernel sorts by length, half of them unknown or with more rows than tokens, rows whose
    magnitudes lie powers of two apart: every row has its own scale."""
    rng = np.random.default_rng(d)
    n, h, g = 240, 2, 4
    lens = [int(x) for x in rng.integers(1, 129, n)]
    cache, codes, scales, tables = filled_cache(M, rng, dev, lens, h, d)
    seqs = [int(x) for x in rng.permutation(n)]
    rows = [min(lens[s], int(rng.integers(1, 90))) for s in seqs]
    for i in range(n):
        if i % 3 == 1:
            seqs[i], rows[i] = (-1 - i if i % 2 else n + i), int(rng.integers(1, 90))
        elif i % 3 == 2 and i % 4 < 2:
            rows[i] = lens[seqs[i]] + int(rng.integers(1, 150))
    t = sum(rows)
    q = rng.normal(0, 1.5, (t, h * g, d)) * np.exp2(rng.integers(-9, 1, (t, h * g, 1)))
    q = torch.from_numpy(q).to(dtype).cuda()
    for _ in range(3):
        out, lse = cache.attend(0, q, i32(seqs), cu_of(rows), max_q=max(rows), return_lse=True)
        check_known(codes[0], scales[0], tables, lens, seqs, rows, q, out, lse)


def huge_pool(cache):
    """The cache said to have 2^24 pages: its tables hold small ones alone, so nothing past its tensors is touched, and
    an image of such a pool (2^24 x 4 kv heads x 64 x 64 x 2 bytes = 550 GB) fits no device."""
    cache._c.pages = 1 << 24
    return cache


def test_failed_scratch_is_no_error_of_the_next_call(M, dev):
    rng = np.random.default_rng(1)
    cache, codes, scales, tables = filled_cache(M, rng, dev, [500] * 4, 2, 64)
    q = torch.from_numpy(rng.normal(0, 1, (2000, 8, 64))).half().cuda()
    small = cache._c.pages
    try:
        huge_pool(cache).attend(0, q, i32(range(4)), cu_of([500] * 4), max_q=500)
    except M.MrlError:
        pass
    cache._c.pages = small
    cache.reserve(i32([1]), i32([3]))
    assert cache.lens.tolist() == [500, 503, 500, 500]


# ---- scratch and captured graphs ------------------------------------------------------------------------------


def reader(M, dev, rng, n, length, h, d, rows, spare=3):
    """A filled cache of n sequences, queries of `rows` rows each, and the call that attends with them."""
    lens = [length] * n
    cache, codes, scales, tables = filled_cache(M, rng, dev, lens, h, d, spare=spare)
    q = torch.from_numpy(rng.normal(0, 1, (n * rows, 4 * h, d))).bfloat16().cuda()
    seqs, cu = i32(range(n)), cu_of([rows] * n)
    return cache, lambda out=None: cache.attend(0, q, seqs, cu, max_q=rows, out=out)


def test_graphs_outlive_growth_and_other_streams(M):
    """Graphs of single rows, of many rows and of a fork, replayed after calls that need more scratch than was there, and
    after calls on more streams than any fixed number of slots."""
    own = M.Device(0)
    rng = np.random.default_rng(2)
    cache1, one = reader(M, own, rng, 8, 3000, 2, 128, 1)
    cache2, many = reader(M, own, rng, 4, 700, 2, 128, 300)
    forks = M.KvCache.create(1, 40, 1, 64, 12, 4, dev=own)
    forks.reserve(i32([0]), i32([150]))
    parents, kids = i32([0] * 8), i32(range(1, 9))
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        own.use_torch_stream()
        want1, want2 = one(), many()
        forks.fork(parents, kids)
        forks.release(kids)
    torch.cuda.synchronize()
    out1, out2 = torch.zeros_like(want1), torch.zeros_like(want2)
    g1, g2, g3 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1, stream=s):
        one(out1)
    with torch.cuda.graph(g2, stream=s):
        many(out2)
    with torch.cuda.graph(g3, stream=s):
        forks.release(kids)
        forks.fork(parents, kids)

    def replayed():
        out1.zero_()
        out2.zero_()
        forks.status.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            for g in (g1, g2, g3):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out1, want1) and torch.equal(out2, want2)
        assert forks.lens.tolist() == [150] * 9 + [0] * 3 and forks.refs.tolist() == [9] * 2 + [1] * 9 + [0] * 29
        assert int(forks.status) == 0

    replayed()
    with torch.cuda.stream(s):
        _, other = reader(M, own, rng, 70, 500, 2, 64, 1)        # another head_dim
        other()
        _, bigger = reader(M, own, rng, 4, 700, 2, 256, 300, spare=400)  # a larger image
        bigger()
        pool = M.KvCache.create(1, 4, 1, 64, 2, 2, dev=own)      # longer lists: a reserve reads refs, tables and lens alone
        refs = torch.zeros(4 << 20, dtype=torch.int32, device="cuda")
        pool._c.refs, pool._c.pages = refs.data_ptr(), refs.shape[0]
        pool.reserve(i32([0]), i32([100]))
        junk = [torch.randn(8 << 20, device="cuda") for _ in range(4)]   # what was freed, if anything was, is used
    torch.cuda.synchronize()
    replayed()
    torch.cuda.synchronize()
    for t in [torch.cuda.Stream() for _ in range(12)]:
        with torch.cuda.stream(t):
            own.use_torch_stream()
            assert torch.equal(one(), want1) and torch.equal(many(), want2)
    torch.cuda.synchronize()
    replayed()
    del g1, g2, g3, junk
    own.close()


def test_growth_during_a_capture_is_refused(M):
    """A capture whose call needs more scratch than there is stays valid: the call is refused before anything is queued."""
    own = M.Device(0)
    rng = np.random.default_rng(3)
    cache, one = reader(M, own, rng, 3, 200, 1, 64, 1)
    s = torch.cuda.Stream()
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        own.use_torch_stream()
        x.add_(1)
        with pytest.raises(M.MrlError, match="capture"):
            one()
    g.replay()
    torch.cuda.synchronize()
    assert x.tolist() == [1.0] * 4
    with torch.cuda.stream(s):
        want = one()
    torch.cuda.synchronize()
    out = torch.zeros_like(want)
    with torch.cuda.graph(g2 := torch.cuda.CUDAGraph(), stream=s):
        one(out)
    g2.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    del g, g2
    own.close()


@pytest.mark.parametrize("d", [64, 256])
def test_many_rows_without_room_for_the_image(M, dev, d):
    """An image that no device has room for: the kernel on the codes gives the same rows."""
    rng = np.random.default_rng(4)
    lens, rows = [700, 64, 300], [500, 64, 300]
    cache, codes, scales, tables = filled_cache(M, rng, dev, lens, 2, d)
    q = torch.from_numpy(rng.normal(0, 1, (sum(rows), 8, d))).bfloat16().cuda()
    out, lse = huge_pool(cache).attend(0, q, i32(range(3)), cu_of(rows), max_q=500, return_lse=True)
    check_known(codes[0], scales[0], tables, lens, range(3), rows, q, out, lse)


# ---- pages that a row does not see ------------------------------------------------------------------------------


def check_by_row(codes, scales, table, n, q, out, lse, window, sinks):
    """One sequence's last rows against the plain form, each row within what the pages that it sees allow: vmax is
    127 times the largest V scale of a page in which the row sees a key."""
    t, hq, d = q.shape
    qn, on, ln = q.double().cpu().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy()
    k, present = held_rows(codes, scales, table, n, 0)
    v, _ = held_rows(codes, scales, table, n, 1)
    want, wl, big = plain_attention(qn, k, v, n - t, True, window, sinks, d ** -0.5, present)
    h = k.shape[1]
    key = np.arange(n)
    for i in range(t):
        p = n - t + i
        ok = present & (key <= p) & ((p - key < window) | (key < sinks) if window else True)
        pages = sorted({int(table[j]) for j in np.nonzero(ok)[0] // PAGE})
        for a in range(h):
            rows = slice(a * hq // h, (a + 1) * hq // h)
            vmax = 127 * float(scales[pages, 1, a].max()) if pages else 0.0
            got, w = on[i, rows], want[i, rows]
            # beyond the output's type the result is its infinity; within a tolerance's width of its end, either
            end, near = float(torch.finfo(q.dtype).max), 0.01 * vmax
            over = np.abs(w) > end - near
            assert np.all((got[over] == np.sign(w[over]) * np.inf) | (np.abs(w[over]) < end + near))
            check_rows(np.where(over, w, got), ln[i, rows], w, wl[i, rows], big, d, n, vmax, U[q.dtype], 2.0 ** -11)


def unseen_scale_case(M, dev, rng, n, t, h, g, d, dtype, window, sinks, pages, ratio, spread=1.0):
    cache, codes, scales, tables = filled_cache(M, rng, dev, [n], h, d)
    for p in pages:
        scales[0, tables[0, p], 1] *= ratio
    cache.scales.copy_(torch.from_numpy(scales))
    q = torch.from_numpy(rng.normal(0, spread, (t, h * g, d))).to(dtype).cuda()
    out, lse = cache.attend(0, q, i32([0]), cu_of([t]), max_q=t, window=window, sinks=sinks, return_lse=True)
    check_by_row(codes[0], scales[0], tables[0], n, q, out, lse, window, sinks)


RATIOS = [1e6, 1e10]


@pytest.mark.parametrize("ratio", RATIOS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_unseen_value_scales_few_rows(M, dev, d, dtype, ratio):
    """A page with far larger values that some rows of a 16-row item see and others do not: a later page (causal), an
    earlier one (window), and one between the sinks and the window."""
    rng = np.random.default_rng(d)
    unseen_scale_case(M, dev, rng, 64 * 3 + 8, 16, 2, 1, d, dtype, 0, 0, [3], ratio)
    unseen_scale_case(M, dev, rng, 64 * 4 + 15, 16, 1, 1, d, dtype, 10, 0, [3], ratio)
    unseen_scale_case(M, dev, rng, 64 * 9 + 20, 12, 2, 2, d, dtype, 6, 4, [1, 8], ratio)
    unseen_scale_case(M, dev, rng, 64 * 40 + 5, 8, 2, 2, d, dtype, 0, 0, [40], ratio)


@pytest.mark.parametrize("ratio", RATIOS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n_seqs", [1, 160])
def test_unseen_value_scales_of_one_warp(M, dev, d, ratio, n_seqs):
    """The first page of a long window, seen by the first four of 16 rows alone and followed by pages of the same warp;
    scores so peaked that a row's result is a few values of a few pages."""
    rng = np.random.default_rng(d + n_seqs)
    n, window, t = 64 * 24 + 11 + 16, 64 * 22 + 16, 16
    assert (n - t - window + 1) % 64 == 60
    lens = [n] * n_seqs
    cache, codes, scales, tables = filled_cache(M, rng, dev, lens, 1, d)
    for i in range(n_seqs):
        scales[0, tables[i, (n - t - window + 1) // 64], 1] *= ratio
    cache.scales.copy_(torch.from_numpy(scales))
    q = torch.from_numpy(rng.normal(0, 8, (n_seqs * t, 1, d))).bfloat16().cuda()
    out, lse = cache.attend(0, q, i32(range(n_seqs)), cu_of([t] * n_seqs), max_q=t, window=window, return_lse=True)
    for i in range(min(n_seqs, 6)):
        rows = slice(i * t, (i + 1) * t)
        check_by_row(codes[0], scales[0], tables[i], n, q[rows], out[rows], lse[rows], window, 0)


@pytest.mark.parametrize("ratio", RATIOS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_unseen_value_scales_many_rows(M, dev, d, dtype, ratio):
    """The same with 128-row tiles: a page that later rows alone see, in either half of a step of 128 keys, pages that
    have left the window, and one between the sinks and the window."""
    rng = np.random.default_rng(d)
    for page in (4, 5):
        unseen_scale_case(M, dev, rng, 700, 660, 2, 4, d, dtype, 0, 0, [page], ratio, spread=5.0)
        unseen_scale_case(M, dev, rng, 700, 700, 1, 8, d, dtype, 40, 0, [page], ratio, spread=5.0)
        unseen_scale_case(M, dev, rng, 900, 600, 2, 4, d, dtype, 70, 4, [1, page], ratio, spread=5.0)


# ---- values that are not finite, windowed attention ---------------------------------------------------------------


def test_redone_rows_do_not_stop_the_call(M, dev):
    """A very long sequence whose last value is not finite: the rows of its last tile that do not see it are computed from
    400,000 keys each, and neither they nor the sequence behind them are given up."""
    rng = np.random.default_rng(6)
    n, m, d = 400000, 300, 64
    q, k, v = (torch.from_numpy(rng.normal(0, 1, (n + m, 1, d)).astype(np.float32)).half().cuda() for _ in range(3))
    v[n - 1, 0, 7] = float("inf")
    out, lse = M.window_attention(q, k, v, i32([0, n, n + m]), max_len=n, causal=True, return_lse=True, dev=dev)
    assert int(dev.attention_status) == 0
    kn, vn = (x[:n - 1, 0].double() for x in (k, v))
    first = n - 400
    s = q[first:n - 1, 0].double() @ kn.T * d ** -0.5
    s.masked_fill_(torch.arange(n - 1, device="cuda") > torch.arange(first, n - 1, device="cuda")[:, None], -math.inf)
    want, wl = torch.softmax(s, 1) @ vn, torch.logsumexp(s, 1)
    big = float((q[first:n - 1, 0].double().abs().max(0).values @ kn.abs().max(0).values) * d ** -0.5)
    check_rows(out[first:n - 1, 0].double().cpu().numpy(), lse[first:n - 1, 0].double().cpu().numpy(), want.cpu().numpy(), wl.cpu().numpy(),
               big, d, n, float(vn.abs().max()), U[q.dtype], U[q.dtype])
    assert float(out[n - 1, 0, 7]) == math.inf and bool(torch.isfinite(out[n - 1, 0, :7]).all())
    qn, kn, vn = (x[n:].double().cpu().numpy() for x in (q, k, v))
    want, wl, big = plain_attention(qn, kn, vn, 0, True, 0, 0, d ** -0.5)
    check_rows(out[n:].double().cpu().numpy(), lse[n:].double().cpu().numpy(), want, wl, big, d, m, np.abs(vn).max(), U[q.dtype], U[q.dtype])


def plain_with_odd_values(q, k, v, causal, window, sinks, scale):
    """plain_attention that keeps what is not visible out of the products: v may hold what is not finite."""
    t, hq, d = q.shape
    h = k.shape[1]
    out = np.zeros((t, hq, d))
    j = np.arange(t)
    for i in range(t):
        ok = np.ones(t, bool)
        if causal:
            ok &= j <= i
        if window:
            ok &= (np.abs(i - j) < window) | (j < sinks)
        for a in range(hq):
            with np.errstate(invalid="ignore"):
                s = k[ok, a // (hq // h)] @ q[i, a] * scale
                w = np.exp(s - s.max())
                out[i, a] = (w / w.sum()) @ v[ok, a // (hq // h)]
    return out


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal,window,sinks", [(True, 0, 0), (True, 60, 4), (False, 0, 0), (False, 90, 2)])
def test_odd_values_seen_and_unseen(M, dev, d, dtype, causal, window, sinks):
    """NaN and both infinities in values at several places, one of them a sink: every column of every row is what its
    visible keys give, NaN and infinity included (weights of these scores are far from 0)."""
    rng = np.random.default_rng(d + window)
    t, h, g = 330, 2, 2
    q, k, v = (torch.from_numpy(rng.normal(0, 0.7, (t, n, d))).to(dtype).cuda() for n in (h * g, h, h))
    nan, inf = float("nan"), float("inf")
    for key, head, dim, x in ((1, 0, 3, inf), (50, 0, 9, nan), (140, 1, 0, -inf), (141, 1, 0, inf), (200, 1, 5, inf), (300, 0, 60, nan)):
        v[key, head, dim] = x
    out = M.window_attention(q, k, v, i32([0, t]), max_len=t, causal=causal, window=window, sinks=sinks, dev=dev).double().cpu().numpy()
    vn = v.double().cpu().numpy()
    want = plain_with_odd_values(q.double().cpu().numpy(), k.double().cpu().numpy(), vn, causal, window, sinks, d ** -0.5)
    assert np.array_equal(np.isnan(want), np.isnan(out))
    odd = ~np.isfinite(want)
    assert np.array_equal(want[odd & ~np.isnan(want)], out[odd & ~np.isnan(want)])
    vmax = np.abs(vn[np.isfinite(vn)]).max()
    check_rows(np.where(odd, 0, out), np.zeros(0), np.where(odd, 0, want), np.zeros(0), 0.0, d, t, vmax, U[dtype], U[dtype])


@pytest.mark.parametrize("where", ["k", "q"])
def test_odd_scores(M, dev, where):
    """A NaN in a key makes every row that sees it NaN, in a query its own row; no other row changes."""
    rng = np.random.default_rng(8)
    t, d = 400, 128
    q, k, v = (torch.from_numpy(rng.normal(0, 1, (t, n, d))).bfloat16().cuda() for n in (4, 2, 2))
    clean, clean_lse = M.window_attention(q, k, v, i32([0, t]), max_len=t, window=100, return_lse=True, dev=dev)
    (k if where == "k" else q)[170, 1] = float("nan")
    out, lse = M.window_attention(q, k, v, i32([0, t]), max_len=t, window=100, return_lse=True, dev=dev)
    rows, heads = (slice(170, 270), slice(2, 4)) if where == "k" else (slice(170, 171), slice(1, 2))
    assert bool(torch.isnan(out[rows, heads]).all()) and bool(torch.isnan(lse[rows, heads]).all())
    out[rows, heads], lse[rows, heads] = clean[rows, heads], clean_lse[rows, heads]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (False, 100)])
def test_rows_behind_a_sequence_do_not_matter(M, dev, d, dtype, causal, window):
    """The rows behind a sequence, those of the next one or none's, hold NaN or Inf: its results keep every bit, as no
    product of theirs meets them (sequences that end at, before and after a step of 128 keys and half of one)."""
    rng = np.random.default_rng(d)
    for n in (1, 60, 64, 65, 127, 128, 129, 190, 193, 400):
        cu = i32([0, n, n + 140])
        q, k, v = (torch.from_numpy(rng.normal(0, 1, (n + 300, x, d))).to(dtype).cuda() for x in (4, 2, 2))
        f = lambda: M.window_attention(q, k, v, cu, max_len=max(n, 140), causal=causal, window=window, return_lse=True, dev=dev)  # noqa: E731
        clean, clean_lse = f()
        for x in (float("nan"), float("inf")):
            for y in (q, k, v):
                y[n:] = x
            out, lse = f()
            assert torch.equal(out[:n], clean[:n]) and torch.equal(lse[:n], clean_lse[:n])


# ---- index tensors whose contents are wrong -----------------------------------------------------------------------


@pytest.mark.parametrize("n_seqs,rows", [(4, 8), (200, 8), (4, 300), (200, 300)])
def test_decreasing_offsets_do_nothing(M, dev, n_seqs, rows):
    """Offsets that decrease give no rows at all, and the status bit: sums over them could leave every range."""
    rng = np.random.default_rng(n_seqs)
    t = n_seqs * rows
    cache, *_ = filled_cache(M, rng, dev, [rows] * n_seqs, 2, 64)
    q, k, v = (torch.from_numpy(rng.normal(0, 1, (t, h, 64)).astype(np.float32)).half().cuda() for h in (4, 2, 2))
    good = cu_of([rows] * n_seqs)
    bad = good.clone()
    bad[2] = 1
    for cu, bits in ((bad, 4), (good, 0)):
        out = torch.full_like(q, 7.0)
        cache.attend(0, q, i32(range(n_seqs)), cu, max_q=rows, out=out)
        assert int(cache.status) == bits and bool((out == 7.0).all()) == (cu is bad)
        out = torch.full_like(q, 7.0)
        M.window_attention(q, k, v, cu, max_len=rows, out=out, dev=dev)
        assert int(dev.attention_status) == bits and bool((out == 7.0).all()) == (cu is bad)
        cache.status.zero_()
        dev.attention_status.zero_()


def test_refused_page_operations_leave_every_length(M, dev):
    """A refused reserve or fork changes nothing, lengths that are none (negative) included."""
    cache = M.KvCache.create(1, 8, 1, 64, 6, 4, dev=dev)
    cache.reserve(i32([0, 1]), i32([70, 10]))
    cache.lens[2], cache.lens[3] = -5, -(1 << 31)
    before = [x.clone() for x in (cache.tables, cache.lens, cache.refs)]
    tried = [lambda: cache.reserve(i32([0, 2]), i32([1, 1])), lambda: cache.reserve(i32([3, 1, 3, 1]), i32([1] * 4)),
             lambda: cache.reserve(i32([4, 4]), i32([1, 1])), lambda: cache.fork(i32([0]), i32([2])),
             lambda: cache.fork(i32([0, 0, 1]), i32([3, 4, 1])), lambda: cache.fork(i32([2]), i32([4])),
             lambda: cache.fork(i32([0, 0]), i32([5, 5]))]
    for f in tried:
        f()
        assert int(cache.status) == 4
        for x, y in zip(before, (cache.tables, cache.lens, cache.refs)):
            assert torch.equal(x, y)
        cache.status.zero_()


def test_rows_that_are_left_out_set_the_status(M, dev):
    """Unknown sequences, more rows than tokens and missing pages: an append, a read and both attention kernels say that
    rows were left out, and the other rows are right."""
    rng = np.random.default_rng(11)
    cache = M.KvCache.create(1, 40, 2, 64, 4, 12, dev=dev)

    def new(t, h=2):
        return torch.from_numpy(rng.normal(0, 1, (t, h, 64)).astype(np.float32)).half().cuda()

    def status():
        s = int(cache.status)
        cache.status.zero_()
        return s

    cache.reserve(i32([0, 1, 2]), i32([100, 300, 10]))
    k = new(410)
    cache.append(0, k, k, i32([0, 1, 2]), cu_of([100, 300, 10]))
    assert status() == 0
    codes, scales = cache.codes.clone(), cache.scales.clone()
    for seqs, rows in (([4], [3]), ([-1], [70]), ([2], [11]), ([3], [1]), ([1 << 30, -5], [1, 1])):
        x = new(sum(rows))
        cache.append(0, x, x, i32(seqs), cu_of(rows))
        assert status() == 4 and torch.equal(codes, cache.codes) and torch.equal(scales, cache.scales)
        got, _ = cache.read(0, i32(seqs), cu_of(rows), tokens=sum(rows))
        assert status() == 4 and not bool(got.any())
    for rows in ([100, 40, 300], [1, 1, 1]):
        q = new(sum(rows), 8)
        out = cache.attend(0, q, i32([0, 1 << 30, 1]), cu_of(rows), max_q=max(rows))
        assert status() == 4
        keep = torch.cat([q[:rows[0]], q[-rows[2]:]])
        assert torch.equal(torch.cat([out[:rows[0]], out[-rows[2]:]]),
                           cache.attend(0, keep, i32([0, 1]), cu_of([rows[0], rows[2]]), max_q=max(rows)))
        assert status() == 0
    assert bool((cache.attend(0, new(3, 8), i32([0, -1, 1]))[1] == 0).all()) and status() == 4
    cache.attend(0, new(12, 8), i32([2]), cu_of([12]), max_q=12)
    assert status() == 4
    # a page that was given back: appended rows that belong there are lost, reads of it are 0 by definition
    cache.trim(i32([1]), 64)
    x = new(300)
    cache.append(0, x, x, i32([1]), cu_of([300]))
    assert status() == 4
    cache.read(0, i32([1]), cu_of([300]), tokens=300)
    assert status() == 0


# ---- refusals ---------------------------------------------------------------------------------------------------------


def test_gradients_are_refused_not_dropped(M, dev):
    """A tensor that requires gradients is refused while they are recorded: the result would be detached without a word."""
    half = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")  # noqa: E731
    cache = M.KvCache.create(1, 4, 2, 64, 3, 2, dev=dev)
    seqs, cu = i32([0, 1]), i32([0, 2])
    cache.reserve(seqs, i32([1, 1]))
    g = half(2, 2, 64).requires_grad_()
    calls = [lambda: cache.append(0, g, half(2, 2, 64), seqs), lambda: cache.append(0, half(2, 2, 64), g, seqs),
             lambda: cache.attend(0, g, seqs), lambda: cache.attend(0, half(2, 2, 64), seqs, out=g),
             lambda: M.window_attention(g, half(2, 2, 64), half(2, 2, 64), cu, 2, dev=dev),
             lambda: M.window_attention(half(2, 2, 64), g, half(2, 2, 64), cu, 2, dev=dev),
             lambda: M.window_attention(half(2, 2, 64), half(2, 2, 64), g, cu, 2, dev=dev)]
    for f in calls:
        with pytest.raises(ValueError, match="gradient"):
            f()
        with torch.no_grad():
            f()
    assert int(cache.status) == 0


def test_read_with_offsets_needs_the_row_count(M, dev):
    """Rows by offsets and no count: the count of sequences stood in for it, and cut the rows short at other positions."""
    cache = M.KvCache.create(1, 8, 1, 64, 2, 4, dev=dev)
    cache.reserve(i32([0, 1]), i32([5, 70]))
    x = torch.randn(75, 1, 64, device="cuda").half()
    cache.append(0, x, x, i32([0, 1]), cu_of([5, 70]))
    with pytest.raises(ValueError, match="tokens"):
        cache.read(0, i32([0, 1]), cu_of([5, 70]))
    with pytest.raises(ValueError, match="tokens"):
        cache.read(0, i32([0, 1]), cu_of([5, 70]), tokens=-1)
    k, _ = cache.read(0, i32([0, 1]), cu_of([5, 70]), tokens=75)
    # half a step of the page's scale, max|x| / 254
    assert float((k - x.float()).abs().max()) <= float(x.float().abs().max()) / 254 * 1.0001
    assert cache.read(0, i32([0, 1]))[0].shape == (2, 1, 64)


@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_strides_beyond_a_tensor_map_name_their_operand(M, dev, name):
    """A row stride of 2^40 bytes, the first that a map cannot hold: refused on the host, by name."""
    from mrl_b200 import attention as A

    x = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
    out, cu = torch.zeros_like(x), i32([0, 2])
    strides = {n: (1 << 39 if n == name else 128, 64) for n in "qkv"}
    M.window_attention(x, x, x, cu, 2, dev=dev)
    args = bytearray(A._ATTN.pack(x.data_ptr(), x.data_ptr(), x.data_ptr(), out.data_ptr(), 0, 0, cu.data_ptr(), 0, *strides["q"], *strides["k"],
                                  *strides["v"], 128, 64, 1, 2, 2, 2, 2, 64, 0, 1, 0, 0, 0.125, 0))
    import ctypes as C

    with pytest.raises(M.MrlError, match=f"^.*\\b{name} has strides"):
        A.check(dev.ptr, dev.lib.mrl_window_attention(dev.ptr, C.addressof((C.c_char * len(args)).from_buffer(args))))
    assert not bool(out.any())


@pytest.mark.parametrize("d", [64, 256])
def test_broadcast_heads_and_rows(M, dev, d):
    """Keys and values of one head shown as several, and values of one row as all: strides of 0, as in an append."""
    rng = np.random.default_rng(d)
    t = 200
    q = torch.from_numpy(rng.normal(0, 1, (t, 4, d)).astype(np.float32)).half().cuda()
    k1, v1 = (torch.from_numpy(rng.normal(0, 1, (t, 1, d)).astype(np.float32)).half().cuda() for _ in range(2))
    k, v, row = k1.expand(t, 2, d), v1.expand(t, 2, d), v1[:1].expand(t, 1, d)
    cu = i32([0, 90, t])
    f = lambda *x: M.window_attention(*x, cu, 110, dev=dev)  # noqa: E731
    assert torch.equal(f(q, k, v), f(q, k.contiguous(), v.contiguous()))
    assert torch.equal(f(q, k1, row), f(q, k1, row.contiguous()))
    q1 = q[:, :1].expand(t, 4, d)
    assert torch.equal(f(q1, k, v), f(q1.contiguous(), k.contiguous(), v.contiguous()))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("h,g", [(1, 4), (2, 3), (3, 1)])
@pytest.mark.parametrize("turned", ["q", "k", "v", "qkv"])
def test_window_heads_outermost(M, dev, d, h, g, turned):
    """Inputs laid out by heads, [heads][rows][dims], each alone and all three: the same bits as laid out by rows."""
    rng = np.random.default_rng(d + h)
    lens = [5, 130, 64, 257]
    t = sum(lens)
    x = {n: torch.from_numpy(rng.normal(0, 1, (t, heads, d)).astype(np.float32)).bfloat16().cuda() for n, heads in (("q", h * g), ("k", h), ("v", h))}
    for causal, window, sinks in ((True, 0, 0), (False, 0, 0), (True, 70, 3), (False, 40, 0)):
        f = lambda y: M.window_attention(y["q"], y["k"], y["v"], cu_of(lens), max_len=max(lens), causal=causal, window=window, sinks=sinks,  # noqa: E731,B023
                                         return_lse=True, dev=dev)
        want, want_lse = f(x)
        y = {n: z.transpose(0, 1).contiguous().transpose(0, 1) if n in turned else z for n, z in x.items()}
        out, lse = f(y)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    qn, kn, vn = (x[n].double().cpu().numpy() for n in "qkv")
    at = 0
    for n in lens:
        want, wl, big = plain_attention(qn[at:at + n], kn[at:at + n], vn[at:at + n], 0, False, 40, 0, d ** -0.5)
        check_rows(out[at:at + n].double().cpu().numpy(), lse[at:at + n].double().cpu().numpy(), want, wl, big, d, n, np.abs(vn[at:at + n]).max(),
                   U[torch.bfloat16], U[torch.bfloat16])
        at += n


# ---- very large values --------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 20, 700])
@pytest.mark.parametrize("n_seqs", [1, 90])
def test_values_near_the_end_of_bf16_over_the_cache(M, dev, d, rows, n_seqs):
    """Values of 1e38, all of one sign in half of the dims: weighted sums of hundreds of them are beyond f32, their means are
    not."""
    if n_seqs * rows > 2000:
        rows = 20
    rng = np.random.default_rng(d)
    n = 700
    cache = M.KvCache.create(1, 11 * n_seqs, 2, d, n_seqs, 11, dev=dev)
    seqs = list(range(n_seqs))
    cache.reserve(i32(seqs), i32([n] * n_seqs))
    k = torch.from_numpy(rng.normal(0, 0.3, (n * n_seqs, 2, d)).astype(np.float32)).bfloat16().cuda()
    v = torch.from_numpy(rng.normal(0, 0.5, (n * n_seqs, 2, d)))
    v[:, :, ::2] = 1 + v[:, :, ::2].abs().clamp(max=1)
    v = (v.clamp(-2, 2) * 1e38).bfloat16().cuda()
    cache.append(0, k, v, i32(seqs), cu_of([n] * n_seqs))
    q = torch.from_numpy(rng.normal(0, 0.5, (rows * n_seqs, 4, d)).astype(np.float32)).bfloat16().cuda()
    out, lse = cache.attend(0, q, i32(seqs), cu_of([rows] * n_seqs), max_q=rows, return_lse=True)
    codes, scales, tables = (x.cpu().numpy() for x in (cache.codes, cache.scales, cache.tables))
    picked = seqs[:3]
    check_known(codes[0], scales[0], tables, [n] * n_seqs, picked, [rows] * len(picked), q, out, lse)
    assert float(out[:, :, ::2].min()) > 0.9e38


def test_values_near_the_end_of_bf16_in_rows(M, dev):
    rng = np.random.default_rng(12)
    n, d = 300, 128
    q, k = (torch.from_numpy(rng.normal(0, 0.5, (n, h, d)).astype(np.float32)).bfloat16().cuda() for h in (4, 2))
    v = (torch.from_numpy(rng.uniform(1, 3, (n, 2, d))) * 1e38).bfloat16().cuda()
    for causal, window in ((True, 0), (False, 0), (True, 100)):
        out, lse = M.window_attention(q, k, v, i32([0, n]), n, causal=causal, window=window, return_lse=True, dev=dev)
        qn, kn, vn = (x.double().cpu().numpy() for x in (q, k, v))
        want, wl, big = plain_attention(qn, kn, vn, 0, causal, window, 0, d ** -0.5)
        check_rows(out.double().cpu().numpy(), lse.double().cpu().numpy(), want, wl, big, d, n, np.abs(vn).max(), U[q.dtype], U[q.dtype])


def test_more_streams_than_scratch_is_kept_for(M):
    """64 streams of one context, twice: some take another's scratch over, a captured graph's never; results and graph stay
    right."""
    own = M.Device(0)
    rng = np.random.default_rng(13)
    _, one = reader(M, own, rng, 8, 3000, 2, 128, 1)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        own.use_torch_stream()
        want = one()
    torch.cuda.synchronize()
    out = torch.zeros_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        one(out)
    streams = [torch.cuda.Stream(priority=-(i % 2)) for i in range(64)]
    assert len({t.cuda_stream for t in streams}) > 40
    free = []
    for _ in range(2):
        for t in streams:
            with torch.cuda.stream(t):
                own.use_torch_stream()
                assert torch.equal(one(), want)
        torch.cuda.synchronize()
        free.append(torch.cuda.mem_get_info()[0])
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert free[0] - free[1] < 64 << 20
    del g
    own.close()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [4, 600])
def test_a_nan_query_is_its_own_rows_matter(M, dev, dtype, rows):
    """Over the cache: a NaN in one head of one row makes that head's row NaN and changes no other bit."""
    rng = np.random.default_rng(14)
    cache, *_ = filled_cache(M, rng, dev, [700, 650], 2, 128)
    q = torch.from_numpy(rng.normal(0, 1, (2 * rows, 8, 128)).astype(np.float32)).to(dtype).cuda()
    f = lambda: cache.attend(0, q, i32([0, 1]), cu_of([rows, rows]), max_q=rows, return_lse=True)  # noqa: E731
    clean, clean_lse = f()
    q[rows + 1, 5, 17] = float("nan")
    out, lse = f()
    assert bool(torch.isnan(out[rows + 1, 5]).all()) and bool(torch.isnan(lse[rows + 1, 5]))
    out[rows + 1, 5], lse[rows + 1, 5] = clean[rows + 1, 5], clean_lse[rows + 1, 5]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)
