"""The paged 8-bit cache, attention over it, and windowed attention over ragged inputs, against plain
implementations in 64 bits (include/mrl_kv.h).

Tolerances. Scores, softmax statistics and sums are kept in f32 and the weights p enter the second
product rounded to 16 bits, so with unit roundoff u (2^-11 for f16, 2^-8 for bf16) a result is off by at
most u_out |o| for its own rounding, u_p sum(p |v|) for the weights', and 2^-25 per key for weights that
are subnormal in f16: (u_out + u_p + n 2^-25) max|v|, with 2e-5 max|v| for the f32 parts. Over the cache
p is f16 (codes are exact in it); over 16-bit inputs it has their type. lse is off by the scores' f32
error, at most 2 D 2^-24 max sum|q k| scale, and 1e-6 (1 + |lse|).
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

PAGE = 64
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def M():
    import mrl_b200

    return mrl_b200


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def cu_of(counts):
    return i32(np.concatenate([[0], np.cumsum(counts)]))


# ---- plain implementations -------------------------------------------------------------------------


def visible(p, n, causal, window, sinks):
    j = np.arange(n)
    ok = np.ones(n, bool)
    if causal:
        ok &= j <= p
    if window:
        ok &= (np.abs(p - j) < window) | (j < sinks)
    return ok


def plain_attention(q, k, v, first, causal, window, sinks, scale, present=None):
    """q [t, hq, d], k, v [n, h, d] float64 numpy, queries at positions first ..; (out, lse, max sum|qk|scale)."""
    t, hq, d = q.shape
    n, h, _ = k.shape
    out, lse, big = np.zeros((t, hq, d)), np.full((t, hq), -np.inf), 0.0
    if t == 0 or n == 0:
        return out, lse, big
    ok = np.stack([visible(first + i, n, causal, window, sinks) for i in range(t)])
    if present is not None:
        ok &= present
    some = ok.any(1)
    for a in range(hq):
        kk, vv = k[:, a // (hq // h)], v[:, a // (hq // h)]
        s = np.where(ok, q[:, a] @ kk.T * scale, -np.inf)
        big = max(big, float(np.where(ok, np.abs(q[:, a]) @ np.abs(kk).T, 0).max() * scale))
        m = np.where(some, s.max(1), 0.0)
        w = np.exp(s - m[:, None])
        total = w.sum(1)
        out[:, a] = w @ vv / np.where(some, total, 1.0)[:, None]
        lse[some, a] = m[some] + np.log(total[some])
    return out, lse, big


def held_rows(codes, scales, table, n, which):
    """The values of K (0) or V (1) of a sequence's first n tokens from one layer's pool (numpy): [n, h, d]
    float64, and which tokens have a page."""
    pages, _, h, block = codes.shape
    d = block // PAGE
    rows, present = np.zeros((n, h, d)), np.zeros(n, bool)
    for i in range((n + PAGE - 1) // PAGE):
        p = int(table[i])
        lo, hi = i * PAGE, min(n, (i + 1) * PAGE)
        if not 0 <= p < pages:
            continue
        c = codes[p, which].astype(np.float64)
        c = c.reshape(h, d // 64, PAGE, 64).transpose(2, 0, 1, 3).reshape(PAGE, h, d) if which == 0 else \
            c.reshape(h, d, PAGE).transpose(2, 0, 1)
        rows[lo:hi] = (c * scales[p, which].astype(np.float64)[None, :, None])[: hi - lo]
        present[lo:hi] = True
    return rows, present


def check_rows(out, lse, want, want_lse, big, d, n, vmax, u_out, u_p):
    tol = (1.05 * (u_out + u_p) + n * 2.0 ** -25 + 2e-5) * vmax + 1e-30
    err = np.abs(out - want).max() if out.size else 0.0
    assert err <= tol, f"out is off by {err:.3g}, at most {tol:.3g}"
    fin = np.isfinite(want_lse)
    assert np.array_equal(fin, np.isfinite(lse))
    assert np.all(lse[~fin] == -np.inf)
    if fin.any():
        e = np.abs(lse[fin] - want_lse[fin])
        lim = 2 * d * 2.0 ** -24 * big + 1e-6 * (1 + np.abs(want_lse[fin]))
        assert np.all(e <= lim), f"lse is off by {e.max():.3g}"


# ---- attention over the cache -------------------------------------------------------------------------


def filled_cache(M, rng, dev, lens, h, d, layers=1, spare=3, width=None):
    """A cache whose sequences hold random codes at random pages; unfilled slots and unused pages hold the
    worst there is: code -128, scale NaN."""
    need = [(n + PAGE - 1) // PAGE for n in lens]
    pages = sum(need) + spare
    width = width or max(need + [1]) + 1
    codes = rng.integers(-127, 128, (layers, pages, 2, h, PAGE * d)).astype(np.int8)
    scales = (np.exp(rng.normal(0, 0.7, (layers, pages, 2, h))) / 60).astype(np.float32)
    order = rng.permutation(pages)
    tables = np.full((len(lens), width), -1, np.int32)
    refs = np.zeros(pages, np.int32)
    at = 0
    for i, m in enumerate(need):
        tables[i, :m] = order[at:at + m]
        refs[order[at:at + m]] = 1
        at += m
        if lens[i] % PAGE:
            tail = codes[:, order[at - 1]]
            tail[:, 0].reshape(layers, h, d // 64, PAGE, 64)[:, :, :, lens[i] % PAGE:] = -128
            tail[:, 1].reshape(layers, h, d, PAGE)[:, :, :, lens[i] % PAGE:] = -128
    scales[:, refs == 0] = np.nan
    cu = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    cache = M.KvCache(cu(codes), cu(scales), cu(tables), i32(lens), cu(refs), dev=dev)
    return cache, codes, scales, tables


def run_attend(M, dev, rng, lens, counts, h, g, d, dtype, window=0, sinks=0, layer=0, layers=1, scale=None, q=None):
    cache, codes, scales, tables = filled_cache(M, rng, dev, lens, h, d, layers)
    order = rng.permutation(len(lens))
    t = int(sum(counts))
    if q is None:
        q = torch.from_numpy(rng.normal(0, 1.5, (t, h * g, d))).to(dtype).cuda()
    by = [counts[i] for i in order]
    out, lse = cache.attend(layer, q, i32(order), cu_of(by), max_q=max(max(counts), 1), window=window, sinks=sinks, scale=scale,
                            return_lse=True)
    verify(cache, codes[layer], scales[layer], tables, lens, order, by, q, out, lse, window, sinks, scale)
    assert int(cache.status) == 0
    return cache, q, order, by, out


def verify(cache, codes, scales, tables, lens, order, by, q, out, lse, window, sinks, scale=None):
    d, dtype = q.shape[2], q.dtype
    qn, on, ln = q.double().cpu().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy()
    at = 0
    for i, m in zip(order, by):
        k, present = held_rows(codes, scales, tables[i], lens[i], 0)
        v, _ = held_rows(codes, scales, tables[i], lens[i], 1)
        want, wl, big = plain_attention(qn[at:at + m], k, v, lens[i] - m, True, window, sinks,
                                        scale if scale is not None else d ** -0.5, present)
        check_rows(on[at:at + m], ln[at:at + m], want, wl, big, d, lens[i], np.abs(v).max() if v.size else 0.0, U[dtype],
                   2.0 ** -11)
        at += m


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("h,g", [(1, 1), (2, 3), (3, 4), (1, 16), (2, 17), (1, 40)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_one_token(M, dev, d, h, g, dtype):
    rng = np.random.default_rng(d * 100 + h * 10 + g)
    lens = [0, 1, 2, 63, 64, 65, 127, 128, 130, 700, 1543]
    run_attend(M, dev, rng, lens, [min(n, 1) for n in lens], h, g, d, dtype)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (64, 0), (65, 64), (100, 4), (300, 70), (5000, 3)])
def test_attend_window(M, dev, d, window, sinks):
    rng = np.random.default_rng(window + sinks)
    lens = [1, 64, 65, 129, 400, 1000]
    run_attend(M, dev, rng, lens, [1] * len(lens), 2, 4, d, torch.bfloat16, window, sinks)
    run_attend(M, dev, rng, lens, [1, 3, 65, 2, 40, 190], 2, 2, d, torch.float16, window, sinks)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("h,g", [(1, 1), (2, 3), (1, 8), (1, 40)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_several_tokens(M, dev, d, h, g, dtype):
    rng = np.random.default_rng(d + h + g)
    lens = [0, 1, 5, 64, 66, 131, 300, 520]
    run_attend(M, dev, rng, lens, [0, 1, 5, 64, 2, 0, 130, 7], h, g, d, dtype)


@pytest.mark.parametrize("n", [1, 3, 70, 400])
def test_attend_batch_sizes(M, dev, n):
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(1, 4000 // n + 70, n)]
    run_attend(M, dev, rng, lens, [1] * n, 2, 4, 64, torch.bfloat16)


def test_attend_one_long_sequence(M, dev):
    run_attend(M, dev, np.random.default_rng(5), [20011], [1], 2, 4, 128, torch.float16)
    run_attend(M, dev, np.random.default_rng(6), [20011], [3], 1, 2, 256, torch.float16, 9000, 5)


def test_attend_layer_and_scale(M, dev):
    run_attend(M, dev, np.random.default_rng(7), [130, 70], [1, 1], 2, 2, 64, torch.float16, layer=2, layers=3, scale=0.31)


def test_attend_large_queries(M, dev):
    """bf16 queries beyond f16's range, against scores of ordinary size (a tiny softmax scale)."""
    rng = np.random.default_rng(8)
    q = (torch.from_numpy(rng.normal(0, 1, (2, 4, 64))) * 3e6).to(torch.bfloat16).cuda()
    run_attend(M, dev, rng, [200, 70], [1, 1], 2, 2, 64, torch.bfloat16, scale=1e-7, q=q)
    q = (torch.from_numpy(rng.normal(0, 1, (40, 4, 128))) * 1e-6).to(torch.bfloat16).cuda()
    run_attend(M, dev, rng, [200], [40], 2, 2, 128, torch.bfloat16, scale=1e5, q=q)


def test_attend_missing_pages(M, dev):
    """Entries that are no page (released, or out of range) hide their keys; a row with no page left is empty."""
    rng = np.random.default_rng(9)
    lens = [64 * 5 + 3, 64 * 4, 130]
    cache, codes, scales, tables = filled_cache(M, rng, dev, lens, 2, 64)
    tables[0, 1], tables[0, 3], tables[1, 2] = -1, 1 << 28, -7
    tables[2, :] = -1
    cache.tables.copy_(torch.from_numpy(tables))
    for counts in ([1, 1, 1], [40, 3, 60]):
        q = torch.from_numpy(rng.normal(0, 1, (sum(counts), 4, 64))).half().cuda()
        out, lse = cache.attend(0, q, i32([0, 1, 2]), cu_of(counts), max_q=max(counts), return_lse=True)
        verify(cache, codes[0], scales[0], tables, lens, [0, 1, 2], counts, q, out, lse, 0, 0)
        assert bool((out[-counts[2]:] == 0).all()) and bool((lse[-counts[2]:] == -math.inf).all())


def test_attend_bad_sequences(M, dev):
    """Sequence numbers out of range, and more rows than a sequence has, give empty rows for the positions
    that do not exist."""
    rng = np.random.default_rng(10)
    cache, codes, scales, tables = filled_cache(M, rng, dev, [70, 2], 1, 64)
    q = torch.from_numpy(rng.normal(0, 1, (4, 2, 64))).half().cuda()
    out, lse = cache.attend(0, q, i32([-1, 0, 2, 1 << 30]), return_lse=True)
    for i in (0, 2, 3):
        assert bool((out[i] == 0).all()) and bool((lse[i] == -math.inf).all())
    assert bool((lse[1] > -math.inf).all())
    out, lse = cache.attend(0, q, i32([1]), cu_of([4]), max_q=4, return_lse=True)
    assert bool((out[:2] == 0).all()) and bool((lse[:2] == -math.inf).all())
    verify(cache, codes[0], scales[0], tables, [70, 2], [1], [2], q[2:], out[2:], lse[2:], 0, 0)


def test_attend_strides_and_out(M, dev):
    rng = np.random.default_rng(11)
    lens, counts = [200, 77, 64], [1, 1, 1]
    cache, codes, scales, tables = filled_cache(M, rng, dev, lens, 2, 128)
    big = torch.from_numpy(rng.normal(0, 1, (3, 9, 136))).half().cuda()
    q = big[:, 1:7, :128][:, :4]
    dst = torch.full((3, 6, 256), 7.0, dtype=torch.float16, device="cuda")
    got, lse = cache.attend(0, q, i32([0, 1, 2]), out=dst[:, 1:5, 64:192], return_lse=True)
    verify(cache, codes[0], scales[0], tables, lens, [0, 1, 2], counts, q, got, lse, 0, 0)
    rest = dst.clone()
    rest[:, 1:5, 64:192] = 7.0
    assert bool((rest == 7.0).all())
    turned = torch.from_numpy(rng.normal(0, 1, (4, 3, 128))).half().cuda().transpose(0, 1)  # heads outermost
    got, lse = cache.attend(0, turned, i32([0, 1, 2]), return_lse=True)
    verify(cache, codes[0], scales[0], tables, lens, [0, 1, 2], counts, turned, got, lse, 0, 0)
    wide = torch.from_numpy(rng.normal(0, 1, (150, 8, 128))).half().cuda()[:, ::2]
    got, lse = cache.attend(0, wide, i32([0]), cu_of([150]), max_q=150, return_lse=True)
    verify(cache, codes[0], scales[0], tables, lens, [0], [150], wide, got, lse, 0, 0)


def test_attend_same_answer_again(M, dev):
    rng = np.random.default_rng(12)
    lens = [int(x) for x in rng.integers(1, 3000, 40)]
    cache, q, order, by, out = run_attend(M, dev, rng, lens, [1] * 40, 2, 4, 128, torch.bfloat16)
    for _ in range(5):
        assert torch.equal(out, cache.attend(0, q, i32(order), cu_of(by), max_q=1))
    assert torch.equal(out, cache.attend(0, q, i32(order)))


def test_attend_on_other_streams(M):
    """A context on its own stream, and calls under several torch streams: ordered with their tensors."""
    own = M.Device(0)
    rng = np.random.default_rng(13)
    lens = [700, 64, 300]
    cache, codes, scales, tables = filled_cache(M, rng, own, lens, 2, 64)
    q0 = torch.from_numpy(rng.normal(0, 1, (3, 4, 64))).half().cuda()
    want = cache.attend(0, q0, i32([0, 1, 2])).clone()
    seqs = i32([0, 1, 2])
    torch.cuda.synchronize()
    for s in [torch.cuda.Stream() for _ in range(10)]:
        with torch.cuda.stream(s):
            big = torch.randn(2048, 2048, device="cuda")
            for _ in range(4):
                big = big @ big * 1e-3
            q = q0 + 0 * big[0, 0].half().nan_to_num()
            got = cache.attend(0, q, seqs)
            same = torch.equal(got, want)
        assert same
    own.use_torch_stream()
    assert torch.equal(cache.attend(0, q0, seqs), want)
    own.set_stream(0)
    assert torch.equal(cache.attend(0, q0, seqs), want)
    torch.cuda.synchronize()
    own.close()


def test_attend_in_a_graph(M, dev):
    rng = np.random.default_rng(14)
    cache, codes, scales, tables = filled_cache(M, rng, dev, [700, 64, 300], 2, 64)
    q, seqs = torch.from_numpy(rng.normal(0, 1, (3, 4, 64))).half().cuda(), i32([0, 1, 2])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        dev.use_torch_stream()
        want = cache.attend(0, q, seqs)
    torch.cuda.synchronize()
    out = torch.zeros_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        cache.attend(0, q, seqs, out=out)
    dev.set_stream(0)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ---- windowed attention over ragged inputs ----------------------------------------------------------------


def run_window(M, dev, rng, lens, h, g, d, dtype, causal, window, sinks, scale=None, poison=None):
    """poison(q, k, v, cu): plants values; the rows in its answer are left out of the comparison."""
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(int)
    t = int(cu[-1])
    q, k, v = (torch.from_numpy(rng.normal(0, s, (t, n, d))).to(dtype).cuda() for s, n in ((1.5, h * g), (1, h), (1, h)))
    qn, kn, vn = (x.double().cpu().numpy() for x in (q, k, v))
    skip = poison(q, k, v, cu) if poison else set()
    out, lse = M.window_attention(q, k, v, i32(cu), max_len=max(max(lens), 1), causal=causal, window=window, sinks=sinks,
                                  scale=scale, return_lse=True, dev=dev)
    on, ln = out.double().cpu().numpy(), lse.double().cpu().numpy()
    for a, b in zip(cu, cu[1:]):
        if a == b:
            continue
        want, wl, big = plain_attention(qn[a:b], kn[a:b], vn[a:b], 0, causal, window, sinks,
                                        scale if scale is not None else d ** -0.5)
        keep = [i for i in range(b - a) if a + i not in skip]
        if keep:
            check_rows(on[a:b][keep], ln[a:b][keep], want[keep], wl[keep], big, d, b - a, np.abs(vn[a:b]).max(), U[dtype], U[dtype])
    return q, k, v, out, lse


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("h,g", [(1, 1), (2, 1), (1, 3), (2, 4), (1, 17), (1, 40)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_window_lengths(M, dev, d, h, g, causal, dtype):
    rng = np.random.default_rng(d + h * 7 + g)
    run_window(M, dev, rng, [1, 0, 2, 63, 64, 65, 127, 128, 129, 0, 200, 300], h, g, d, dtype, causal, 0, 0)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (33, 0), (128, 4), (129, 130), (1000, 2)])
def test_window_masks(M, dev, d, causal, window, sinks):
    rng = np.random.default_rng(window)
    run_window(M, dev, rng, [5, 130, 400, 257], 2, 2, d, torch.float16, causal, window, sinks)
    run_window(M, dev, rng, [900], 1, 4, d, torch.bfloat16, causal, window, sinks)


def test_window_one_long_sequence(M, dev):
    run_window(M, dev, np.random.default_rng(1), [1500, 1], 1, 2, 128, torch.bfloat16, True, 0, 0)
    run_window(M, dev, np.random.default_rng(2), [1500, 1], 1, 2, 128, torch.bfloat16, False, 200, 3, scale=0.2)


def test_window_growing_scores(M, dev):
    """Scores that grow along the keys, so that the running maximum moves at every tile."""
    rng = np.random.default_rng(3)
    t, d = 1000, 64
    q = torch.ones(t, 2, d, dtype=torch.float16, device="cuda")
    k = (torch.linspace(0, 6, t)[:, None, None] * torch.ones(t, 1, d)).half().cuda()
    v = torch.from_numpy(rng.normal(0, 1, (t, 1, d))).half().cuda()
    for causal in (True, False):
        for sign in (1.0, -1.0):
            out, lse = M.window_attention(q, k * sign, v, i32([0, t]), max_len=t, causal=causal, return_lse=True, dev=dev)
            kn, vn = (k * sign).double().cpu().numpy(), v.double().cpu().numpy()
            want, wl, big = plain_attention(q.double().cpu().numpy(), kn, vn, 0, causal, 0, 0, d ** -0.5)
            check_rows(out.double().cpu().numpy(), lse.double().cpu().numpy(), want, wl, big, d, t, np.abs(vn).max(), U[q.dtype], U[q.dtype])


@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_window_keys_not_seen(M, dev, what, d):
    """NaN and Inf in one sequence reach neither its neighbours nor the rows that do not see their key."""
    rng = np.random.default_rng(4)

    def first_of_second(q, k, v, cu):
        k[cu[1]:cu[2]] = what
        v[cu[1]:cu[2]] = what
        q[cu[1]:cu[2]] = what
        return set(range(cu[1], cu[2]))

    for dtype in (torch.float16, torch.bfloat16):
        run_window(M, dev, rng, [70, 30, 150, 200], 1, 2, d, dtype, False, 0, 0, poison=first_of_second)

        def late_key(q, k, v, cu):  # causal, window 50: key 100 is seen by rows 100 .. 149 alone
            k[100] = what
            v[100] = what
            return set(range(100, 150))

        run_window(M, dev, rng, [300], 2, 2, d, dtype, True, 50, 0, poison=late_key)

        def mid_key(q, k, v, cu):  # both directions, window 50: rows 151 .. 249 alone
            v[200] = what
            return set(range(151, 250))

        run_window(M, dev, rng, [400], 2, 1, d, dtype, False, 50, 3, poison=mid_key)


def test_window_nonfinite_values_that_are_seen(M, dev):
    """A row that sees a NaN value has a NaN there and nowhere else."""
    rng = np.random.default_rng(5)
    q, k, v = (torch.from_numpy(rng.normal(0, 1, (200, 1, 64))).half().cuda() for _ in range(3))
    v[60, 0, 5] = float("nan")
    out = M.window_attention(q, k, v, i32([0, 200]), max_len=200, causal=True, dev=dev)
    bad = torch.isnan(out)
    assert bool(bad[60:, 0, 5].all()) and int(bad.sum()) == 140


def test_window_strides(M, dev):
    rng = np.random.default_rng(6)
    t, d = 210, 64
    qkv = torch.from_numpy(rng.normal(0, 1, (t, 4 + 2 * 2, d))).half().cuda()
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    turned = torch.empty(4, t, d, dtype=torch.float16, device="cuda").transpose(0, 1)
    a = M.window_attention(q, k, v, i32([0, 100, t]), max_len=110, causal=False, out=turned, dev=dev)
    b = M.window_attention(q.contiguous(), k.contiguous(), v.contiguous(), i32([0, 100, t]), max_len=110, causal=False, dev=dev)
    assert torch.equal(a, b)


# ---- appends ----------------------------------------------------------------------------------------------


class HostCache:
    """The cache's rules on the host, in f32 where they say f32."""

    def __init__(self, layers, pages, h, d, max_seqs, max_pages):
        self.codes = np.zeros((layers, pages, 2, h, PAGE * d), np.int8)
        self.scales = np.zeros((layers, pages, 2, h), np.float32)
        self.tables = np.full((max_seqs, max_pages), -1, np.int32)
        self.lens = np.zeros(max_seqs, np.int32)
        self.refs = np.zeros(pages, np.int32)
        self.h, self.d, self.max_pages = h, d, max_pages
        self.status = 0

    def free(self):
        return [int(p) for p in np.nonzero(self.refs == 0)[0]]

    def reserve(self, seqs, add):
        plan, free = [], self.free()
        for s, a in zip(seqs, add):
            if not 0 <= s < len(self.lens) or a < 0 or list(seqs).count(s) > 1:
                self.status |= 4
                return
        for s, a in zip(seqs, add):
            if (self.lens[s] + a + PAGE - 1) // PAGE > self.max_pages:
                self.status |= 2
                return
            for i in range((self.lens[s] + PAGE - 1) // PAGE, (self.lens[s] + a + PAGE - 1) // PAGE):
                plan.append((s, i))
        if len(plan) > len(free):
            self.status |= 1
            return
        for (s, i), p in zip(plan, free):
            self.tables[s, i] = p
            self.refs[p] = 1
        for s, a in zip(seqs, add):
            self.lens[s] += a

    def release(self, seqs):
        for s in seqs:
            for p in self.tables[s]:
                if p >= 0:
                    self.refs[p] -= 1
            self.tables[s] = -1
            self.lens[s] = 0

    def trim(self, seqs, window, sinks):
        for s in seqs:
            for i in range((self.lens[s] + PAGE - 1) // PAGE):
                first_kept = max(0, self.lens[s] - window + 1)
                if i * PAGE >= sinks and (i + 1) * PAGE <= first_kept and self.tables[s, i] >= 0:
                    self.refs[self.tables[s, i]] -= 1
                    self.tables[s, i] = -1

    def copy(self, src, dst):
        self.codes[:, dst] = self.codes[:, src]
        self.scales[:, dst] = self.scales[:, src]

    def fork(self, parents, children):
        for p, c in zip(parents, children):
            ok = 0 <= p < len(self.lens) and 0 <= c < len(self.lens)
            if not ok or self.lens[c] or not self.lens[p] or list(children).count(c) > 1:
                self.status |= 4
                return
        tails = [(p, c) for p, c in zip(parents, children) if self.lens[p] % PAGE and self.tables[p, self.lens[p] // PAGE] >= 0]
        free = self.free()
        if len(tails) > len(free):
            self.status |= 1
            return
        own = {c: f for (_, c), f in zip(tails, free)}
        for p, c in zip(parents, children):
            full = self.lens[p] // PAGE
            self.tables[c, :full] = self.tables[p, :full]
            for x in self.tables[p, :full]:
                if x >= 0:
                    self.refs[x] += 1
            if c in own:
                self.tables[c, full] = own[c]
                self.refs[own[c]] = 1
                self.copy(self.tables[p, full], own[c])
            self.lens[c] = self.lens[p]

    def compact(self):
        live = int((self.refs > 0).sum())
        holes = [p for p in range(live) if self.refs[p] == 0]
        highs = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        for to, at in zip(holes, highs):
            self.copy(at, to)
            self.refs[to], self.refs[at] = self.refs[at], 0
            self.tables[self.tables == at] = to

    def append(self, layer, k, v, seqs, counts):
        f = np.float32
        at = 0
        for s, m in zip(seqs, counts):
            pos = int(self.lens[s]) - m
            while pos < self.lens[s]:
                end = min(int(self.lens[s]), (pos // PAGE + 1) * PAGE)
                page, slot = self.tables[s, pos // PAGE], pos % PAGE
                for which, x in ((0, k), (1, v)):
                    x = x[at:at + end - pos]
                    fine = np.where(np.isfinite(x), x, f(0))
                    for a in range(self.h):
                        top = f(np.abs(fine[:, a]).max())
                        old, new = self.scales[layer, page, which, a], f(top * f(1.0 / 127.0))
                        block = self.codes[layer, page, which, a]
                        if slot:
                            new = old if top <= f(f(127) * old) else max(new, f(f(2) * old))
                            if new > old:
                                block[:] = np.rint(block.astype(f) * f(old / new)).astype(np.int8)
                        self.scales[layer, page, which, a] = new
                        with np.errstate(invalid="ignore", divide="ignore"):
                            c = np.rint(x[:, a] / new) if new > 0 else np.zeros_like(x[:, a])
                        c = np.clip(np.where(np.isnan(c), 0, c), -127, 127).astype(np.int8)
                        if which == 0:
                            block.reshape(self.d // 64, PAGE, 64)[:, slot:slot + end - pos] = c.reshape(-1, self.d // 64, 64).transpose(1, 0, 2)
                        else:
                            block.reshape(self.d, PAGE)[:, slot:slot + end - pos] = c.T
                at += end - pos
                pos = end


def pair(M, dev, layers, pages, h, d, max_seqs, max_pages):
    return M.KvCache.create(layers, pages, h, d, max_seqs, max_pages, dev=dev), HostCache(layers, pages, h, d, max_seqs, max_pages)


def same(cache, host):
    for name in ("tables", "lens", "refs", "scales", "codes"):
        got, want = getattr(cache, name).cpu().numpy(), getattr(host, name)
        assert np.array_equal(got, want), f"{name} differ at {np.argwhere(got != want)[:4].tolist()}"
    assert int(cache.status) & ~8 == host.status


def append_both(cache, host, rng, layer, seqs, counts, dtype, strange=False):
    t = int(sum(counts))
    both = (rng.normal(0, 1, (t, 2, host.h, host.d)) * np.exp(rng.normal(0, 1, (1, 2, host.h, 1)))).astype(np.float32)
    x = torch.from_numpy(both).to(dtype)
    if strange and t:
        x[rng.integers(t), 0, 0, 3] = float("nan")
        x[rng.integers(t), 1, -1, 5] = float("inf")
        x[rng.integers(t), 0, -1, 7] = -float("inf")
        x[rng.integers(t), 1] = 0
    xc = x.cuda()
    cache.append(layer, xc[:, 0], xc[:, 1], i32(seqs), cu_of(counts))
    xn = x.float().numpy()
    host.append(layer, xn[:, 0], xn[:, 1], seqs, counts)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h", [1, 3])
def test_append(M, dev, d, dtype, h):
    """Codes and scales bit for bit over rounds of appends: single tokens, chunks that cross pages, zero rows."""
    rng = np.random.default_rng(d + h)
    cache, host = pair(M, dev, 2, 40, h, d, 6, 12)
    for step, counts in enumerate([[1, 64, 63, 0, 200], [1, 1, 1, 1, 1], [62, 0, 1, 5, 65], [1, 1, 1, 1, 1], [130, 3, 0, 64, 128]]):
        seqs = [4, 0, 5, 2, 1]
        cache.reserve(i32(seqs), i32(counts))
        host.reserve(seqs, counts)
        for layer in (0, 1):
            append_both(cache, host, rng, layer, seqs, counts, dtype, strange=step == 3)
        same(cache, host)
        k, v = cache.read(1, i32(seqs), cu_of(counts), tokens=sum(counts))
        at = 0
        for s, m in zip(seqs, counts):
            for which, got in ((0, k), (1, v)):
                rows, _ = held_rows(host.codes[1], host.scales[1], host.tables[s], int(host.lens[s]), which)
                want = rows[int(host.lens[s]) - m:].astype(np.float32)
                assert np.array_equal(got[at:at + m].cpu().numpy(), want)
            at += m
    assert int(cache.status) == 8  # the strange values were seen
    k16, _ = cache.read(1, i32(seqs), cu_of(counts), tokens=sum(counts), dtype=dtype)
    assert torch.equal(k16, k.to(dtype))


def test_append_one_row_each(M, dev):
    rng = np.random.default_rng(3)
    cache, host = pair(M, dev, 1, 30, 2, 64, 20, 2)
    seqs = [int(x) for x in rng.permutation(20)]
    for _ in range(70):
        cache.reserve(i32(seqs[:7]), i32([1] * 7))
        host.reserve(seqs[:7], [1] * 7)
        x = torch.from_numpy(rng.normal(0, 1, (7, 2, 2, 64)) * np.exp(rng.normal(0, 2))).half()
        xc = x.cuda()
        cache.append(0, xc[:, 0], xc[:, 1], i32(seqs[:7]))
        host.append(0, x[:, 0].float().numpy(), x[:, 1].float().numpy(), seqs[:7], [1] * 7)
    same(cache, host)


def test_append_rounding_stays_small(M, dev):
    """Tokens appended one at a time with growing magnitudes: the oldest are still within 1.5 steps of the
    page's final scale (half a step of their own rounding, under one step of all later ones together)."""
    cache = M.KvCache.create(1, 1, 1, 64, 1, 1, dev=dev)
    rng = np.random.default_rng(4)
    rows = (rng.normal(0, 1, (64, 1, 64)) * np.linspace(0.1, 30, 64)[:, None, None]).astype(np.float16)
    for i in range(64):
        cache.reserve(i32([0]), i32([1]))
        x = torch.from_numpy(rows[i:i + 1]).cuda()
        cache.append(0, x, x, i32([0]))
    k, v = cache.read(0, i32([0]), cu_of([64]), tokens=64)
    for got, which in ((k, 0), (v, 1)):
        step = float(cache.scales[0, 0, which, 0])
        assert np.abs(got.cpu().numpy().astype(np.float64) - rows.astype(np.float64)).max() <= 1.5 * step


def test_append_then_attend_is_attention(M, dev):
    """The cache against attention over the 16-bit values it was given: within what 8 bits allow. A value
    is off by at most half a step, s/2 = max|x| / 254 per page: scores by sum|q| max|k| / 254 scale = e,
    weights by exp(2 e), so the result by max|v| (1/254 + 2 (exp(2 e) - 1)) and 16-bit roundings."""
    rng = np.random.default_rng(5)
    d, h, g, n = 64, 2, 2, 333
    cache = M.KvCache.create(1, 8, h, d, 1, 8, dev=dev)
    k, v = (torch.from_numpy(rng.normal(0, 1, (n, h, d))).half().cuda() for _ in range(2))
    q = torch.from_numpy(rng.normal(0, 0.2, (n, h * g, d))).half().cuda()
    cache.reserve(i32([0]), i32([n]))
    cache.append(0, k, v, i32([0]), cu_of([n]))
    a = cache.attend(0, q, i32([0]), cu_of([n]), max_q=n).double()
    b = M.window_attention(q, k, v, i32([0, n]), max_len=n, dev=dev).double()
    e = float(q.double().abs().sum(-1).max() * k.abs().max().double() / 254 * d ** -0.5)
    vmax = float(v.abs().max())
    assert float((a - b).abs().max()) <= vmax * (1 / 254 + 2 * (math.exp(2 * e) - 1) + 4 * 2.0 ** -11)


# ---- pages ------------------------------------------------------------------------------------------------


def test_pages_random_walk(M, dev):
    """300 random page operations and appends against the host's rules, everything equal after each."""
    rng = np.random.default_rng(6)
    cache, host = pair(M, dev, 2, 50, 1, 64, 12, 9)
    kinds = set()
    for step in range(300):
        live = [s for s in range(12) if host.lens[s]]
        empty = [s for s in range(12) if not host.lens[s]]
        op = rng.choice(["reserve", "reserve", "fork", "fork", "release", "trim", "compact"])
        if op == "reserve":
            seqs = [int(s) for s in rng.permutation(12)[:rng.integers(1, 5)]]
            add = [int(x) for x in rng.integers(0, 150, len(seqs))]
            before = host.lens.copy()
            cache.reserve(i32(seqs), i32(add))
            host.reserve(seqs, add)
            if not np.array_equal(before, host.lens):
                # appends write a trimmed tail nowhere, as the host's would fault there: rows with pages only
                ok = [(s, a) for s, a in zip(seqs, add) if a and all(
                    host.tables[s, i] >= 0 for i in range((host.lens[s] - a) // PAGE, (host.lens[s] + PAGE - 1) // PAGE))]
                if ok:
                    append_both(cache, host, rng, int(rng.integers(2)), [s for s, _ in ok], [a for _, a in ok], torch.float16)
        elif op == "fork" and live and empty:
            n = int(rng.integers(1, len(empty) + 1))
            parents = [int(rng.choice(live)) for _ in range(n)]
            children = empty[:n]
            cache.fork(i32(parents), i32(children))
            host.fork(parents, children)
        elif op == "release" and live:
            seqs = [int(s) for s in rng.permutation(live)[:rng.integers(1, 4)]]
            cache.release(i32(seqs))
            host.release(seqs)
        elif op == "trim" and live:
            seqs = [int(rng.choice(live))]
            window, sinks = int(rng.integers(1, 300)), int(rng.integers(0, 130))
            cache.trim(i32(seqs), window, sinks)
            host.trim(seqs, window, sinks)
        elif op == "compact":
            cache.compact()
            host.compact()
        else:
            continue
        kinds.add(op)
        same(cache, host)
        cache.status.zero_()
        host.status = 0
    assert kinds == {"reserve", "fork", "release", "trim", "compact"}


def test_pages_large_pool(M, dev):
    """A pool of more pages than one step of the plan covers, with holes everywhere."""
    rng = np.random.default_rng(7)
    cache, host = pair(M, dev, 1, 40000, 1, 64, 900, 60)
    add = [int(x) for x in rng.integers(1, 3600, 900)]
    cache.reserve(i32(range(900)), i32(add))
    host.reserve(list(range(900)), add)
    gone = [int(s) for s in rng.permutation(900)[:500]]
    cache.release(i32(gone))
    host.release(gone)
    same(cache, host)
    cache.codes.random_(-127, 128)
    cache.scales.uniform_()
    host.codes, host.scales = cache.codes.cpu().numpy(), cache.scales.cpu().numpy()
    cache.compact()
    host.compact()
    same(cache, host)
    left = sorted(set(range(900)) - set(gone))
    parents = [left[i % len(left)] for i in range(500)]
    cache.fork(i32(parents), i32(gone))
    host.fork(parents, gone)
    same(cache, host)


def test_pages_refused(M, dev):
    """What cannot be done sets its bit and changes nothing."""
    cache, host = pair(M, dev, 1, 6, 1, 64, 5, 4)

    def tried(bit, f):
        before = [x.clone() for x in (cache.tables, cache.lens, cache.refs)]
        cache.status.zero_()
        f()
        assert int(cache.status) == bit
        for x, y in zip(before, (cache.tables, cache.lens, cache.refs)):
            assert torch.equal(x, y)
        cache.status.zero_()

    cache.reserve(i32([0, 1]), i32([100, 64]))
    tried(1, lambda: cache.reserve(i32([2, 3]), i32([128, 129])))      # 3 pages left, 5 wanted
    tried(2, lambda: cache.reserve(i32([2]), i32([64 * 4 + 1])))
    tried(4, lambda: cache.reserve(i32([2, 5]), i32([1, 1])))
    tried(4, lambda: cache.reserve(i32([2, -1]), i32([1, 1])))
    tried(4, lambda: cache.reserve(i32([2]), i32([-1])))
    tried(4, lambda: cache.reserve(i32([2, 3, 2]), i32([1, 1, 1])))
    tried(4, lambda: cache.fork(i32([0, 0]), i32([2, 1])))              # 1 is not empty
    tried(4, lambda: cache.fork(i32([0, 0]), i32([2, 2])))
    tried(4, lambda: cache.fork(i32([0, 2]), i32([2, 3])))              # 2 is empty, and a child
    tried(4, lambda: cache.fork(i32([0, 9]), i32([2, 3])))
    tried(4, lambda: cache.fork(i32([0]), i32([0])))
    tried(4, lambda: cache.release(i32([7])))
    tried(4, lambda: cache.copy_pages(i32([0]), i32([6])))
    cache.reserve(i32([4]), i32([64 * 3]))
    tried(1, lambda: cache.fork(i32([0]), i32([2])))                    # no page for the tail
    cache.release(i32([4, 4, 4]))                                       # listed twice: given back once
    assert cache.refs.tolist() == [1, 1, 1, 0, 0, 0]


def test_copy_pages(M, dev):
    rng = np.random.default_rng(8)
    cache, host = pair(M, dev, 3, 9, 2, 128, 2, 2)
    cache.codes.random_(-127, 128)
    cache.scales.uniform_()
    host.codes, host.scales = cache.codes.cpu().numpy(), cache.scales.cpu().numpy()
    cache.copy_pages(i32([0, 5, 0]), i32([3, 8, 7]))
    for a, b in ((0, 3), (5, 8), (0, 7)):
        host.copy(a, b)
    same(cache, host)


# ---- refusals ---------------------------------------------------------------------------------------------


def test_refusals(M, dev):
    cache = M.KvCache.create(2, 4, 2, 64, 3, 2, dev=dev)
    half = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")  # noqa: E731
    seqs = i32([0, 1])
    bad = [
        lambda: M.KvCache.create(1, 4, 2, 96, 3, 2, dev=dev),
        lambda: M.KvCache.create(0, 4, 2, 64, 3, 2, dev=dev),
        lambda: M.KvCache(cache.codes, cache.scales[:1], cache.tables, cache.lens, cache.refs, dev=dev),
        lambda: M.KvCache(cache.codes.view(torch.uint8), cache.scales, cache.tables, cache.lens, cache.refs, dev=dev),
        lambda: M.KvCache(cache.codes, cache.scales, cache.tables, cache.lens[:2], cache.refs, dev=dev),
        lambda: cache.reserve(seqs, i32([1])),
        lambda: cache.reserve(seqs.long(), seqs),
        lambda: cache.reserve(seqs.cpu(), seqs),
        lambda: cache.fork(seqs, i32([2])),
        lambda: cache.trim(seqs, -1),
        lambda: cache.append(0, half(2, 2, 64), half(2, 2, 64).bfloat16(), seqs),
        lambda: cache.append(0, half(2, 2, 64).float(), half(2, 2, 64).float(), seqs),
        lambda: cache.append(0, half(2, 3, 64), half(2, 3, 64), seqs),
        lambda: cache.append(0, half(3, 2, 64), half(3, 2, 64), seqs),
        lambda: cache.append(0, half(2, 64, 2).transpose(1, 2), half(2, 2, 64), seqs),
        lambda: cache.attend(0, half(2, 4, 128), seqs),
        lambda: cache.attend(0, half(3, 4, 64), seqs),
        lambda: cache.attend(0, half(2, 4, 64), seqs, i32([0, 2])),
        lambda: cache.attend(0, half(2, 4, 64), seqs, window=-1),
        lambda: cache.attend(0, half(2, 4, 64), seqs, out=half(2, 4, 128)),
        lambda: cache.read(0, seqs, tokens=3),
        lambda: cache.read(0, seqs, dtype=torch.int32),
        lambda: M.window_attention(half(4, 2, 64), half(3, 2, 64), half(3, 2, 64), i32([0, 4]), 4, dev=dev),
        lambda: M.window_attention(half(4, 2, 64), half(4, 2, 64), half(4, 1, 64), i32([0, 4]), 4, dev=dev),
        lambda: M.window_attention(half(4, 2, 64).cpu(), half(4, 2, 64), half(4, 2, 64), i32([0, 4]), 4, dev=dev),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was accepted")
    refused = [
        (lambda: cache.attend(2, half(2, 4, 64), seqs), "layer"),
        (lambda: cache.append(9, half(2, 2, 64), half(2, 2, 64), seqs), "layer"),
        (lambda: cache.attend(0, half(2, 3, 64), seqs), "q_heads"),
        (lambda: cache.attend(0, half(2, 130, 64), seqs), "q_heads"),
        (lambda: cache.attend(0, half(2, 4, 64), seqs, scale=0.0), "scale"),
        (lambda: cache.attend(0, half(2, 4, 64), seqs, scale=float("nan")), "scale"),
        (lambda: cache.attend(0, half(2, 4, 64), seqs, max_q=0), "max_rows"),
        (lambda: cache.attend(0, half(2, 4, 68)[:, :, 2:66], seqs), "multiples of 16 bytes"),
        (lambda: cache.trim(seqs, 0), "window"),
        (lambda: M.window_attention(half(4, 2, 96), half(4, 2, 96), half(4, 2, 96), i32([0, 4]), 4, dev=dev), "head_dim"),
        (lambda: M.window_attention(half(4, 3, 64), half(4, 2, 64), half(4, 2, 64), i32([0, 4]), 4, dev=dev), "q_heads"),
        (lambda: M.window_attention(half(4, 2, 64), half(4, 2, 64), half(4, 2, 64), i32([0, 4]), 0, dev=dev), "max_rows"),
        (lambda: M.window_attention(half(4, 2, 64), half(4, 2, 64), half(4, 2, 64), i32([0]), 4, dev=dev), "no sequences"),
    ]
    for f, word in refused:
        with pytest.raises(M.MrlError, match=word):
            f()
    # nothing to do is not an error
    none = i32([])
    cache.reserve(none, none)
    cache.fork(none, none)
    cache.release(none)
    cache.append(0, half(0, 2, 64), half(0, 2, 64), none)
    assert cache.attend(0, half(0, 4, 64), none).shape == (0, 4, 64)
    assert cache.read(0, none)[0].shape == (0, 2, 64)
    assert M.window_attention(half(0, 2, 64), half(0, 2, 64), half(0, 2, 64), i32([0]), 0, dev=dev).shape == (0, 2, 64)
    assert int(cache.status) == 0


# ---- attention of many rows over the cache (the pages widened first, 128-row tiles) ------------------------------

MANY_LENS = [0, 1, 5, 64, 66, 131, 300, 520, 900, 1300]
MANY_ROWS = [0, 1, 5, 64, 2, 0, 300, 400, 900, 1000]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("h,g,window,sinks", [(2, 4, 0, 0), (4, 3, 0, 0), (2, 4, 100, 70), (1, 17, 33, 0), (3, 4, 400, 4), (8, 1, 1, 1)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_many_rows(M, dev, d, h, g, window, sinks, dtype):
    rng = np.random.default_rng(d + h + g + window)
    run_attend(M, dev, rng, MANY_LENS, MANY_ROWS, h, g, d, dtype, window, sinks)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_many_rows_missing_pages(M, dev, d):
    """Pages that are gone in the middle, out-of-range entries, a sequence without any, sequences out of range."""
    rng = np.random.default_rng(d)
    cache, codes, scales, tables = filled_cache(M, rng, dev, MANY_LENS, 2, d)
    tables[9, 1], tables[9, 4], tables[8, 2], tables[8, 3] = -1, 1 << 28, -7, -1
    tables[6, :] = -1
    cache.tables.copy_(torch.from_numpy(tables))
    q = torch.from_numpy(rng.normal(0, 1, (sum(MANY_ROWS), 8, d))).half().cuda()
    out, lse = cache.attend(0, q, i32(range(10)), cu_of(MANY_ROWS), max_q=1000, return_lse=True)
    verify(cache, codes[0], scales[0], tables, MANY_LENS, range(10), MANY_ROWS, q, out, lse, 0, 0)
    seqs = list(range(10))
    seqs[9], seqs[7] = -1, 1 << 30
    out2, lse2 = cache.attend(0, q, i32(seqs), cu_of(MANY_ROWS), max_q=1000, return_lse=True)
    cu = np.concatenate([[0], np.cumsum(MANY_ROWS)])
    for i in (7, 9):
        assert bool((out2[cu[i]:cu[i + 1]] == 0).all()) and bool((lse2[cu[i]:cu[i + 1]] == -math.inf).all())
    assert torch.equal(out2[cu[8]:cu[9]], out[cu[8]:cu[9]])


def test_attend_many_rows_shared_pages(M, dev):
    """Forks: a prefix that many sequences share is widened once, their own tails each."""
    rng = np.random.default_rng(21)
    n, h, g, d = 40, 2, 4, 64
    cache = M.KvCache.create(2, 120, h, d, n + 1, 8, dev=dev)

    def extend(seqs, counts):
        cache.reserve(i32(seqs), i32(counts))
        for layer in range(2):
            kv = torch.from_numpy(rng.normal(0, 1, (sum(counts), 2, h, d))).half().cuda()
            cache.append(layer, kv[:, 0], kv[:, 1], i32(seqs), cu_of(counts))

    extend([0], [150])
    kids = list(range(1, n + 1))
    cache.fork(i32([0] * n), i32(kids))
    counts = [int(x) for x in rng.integers(20, 100, n)]
    extend(kids, counts)
    assert int(cache.refs.max()) == n + 1
    q = torch.from_numpy(rng.normal(0, 1, (sum(counts), h * g, d))).half().cuda()
    for layer in range(2):
        out, lse = cache.attend(layer, q, i32(kids), cu_of(counts), max_q=100, return_lse=True)
        verify(cache, cache.codes[layer].cpu().numpy(), cache.scales[layer].cpu().numpy(), cache.tables.cpu().numpy(),
               [int(x) for x in cache.lens], kids, counts, q, out, lse, 0, 0)


def test_attend_many_rows_again_and_strided(M, dev):
    rng = np.random.default_rng(22)
    cache, codes, scales, tables = filled_cache(M, rng, dev, MANY_LENS, 2, 128)
    wide = torch.from_numpy(rng.normal(0, 1, (sum(MANY_ROWS), 17, 128))).bfloat16().cuda()[:, 1::2]
    dst = torch.full((sum(MANY_ROWS), 9, 136), 7.0, dtype=torch.bfloat16, device="cuda")
    out, lse = cache.attend(0, wide, i32(range(10)), cu_of(MANY_ROWS), max_q=1000, out=dst[:, 1:, :128], return_lse=True)
    verify(cache, codes[0], scales[0], tables, MANY_LENS, range(10), MANY_ROWS, wide, out, lse, 0, 0)
    assert bool((dst[:, 0] == 7.0).all()) and bool((dst[:, :, 128:] == 7.0).all())
    first = out.clone()
    for _ in range(4):
        assert torch.equal(first, cache.attend(0, wide, i32(range(10)), cu_of(MANY_ROWS), max_q=1000))


def test_attend_more_sequences_than_a_launch_holds(M, dev):
    """1,300 sequences of one row and of several: more than one launch's table of sequences."""
    rng = np.random.default_rng(23)
    lens = [int(x) for x in rng.integers(1, 90, 1300)]
    run_attend(M, dev, rng, lens, [1] * 1300, 1, 2, 64, torch.float16)
    run_attend(M, dev, rng, lens, [min(x, 40) for x in lens], 1, 8, 64, torch.float16)
    run_window(M, dev, rng, lens, 1, 2, 64, torch.float16, True, 0, 0)
