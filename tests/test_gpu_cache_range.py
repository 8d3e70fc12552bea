"""GPU: the paged K/V cache where values and numbers are far from ordinary ones: rows of very different sizes, zeros, NaN
alone in a tile, large values of V, batches whose numbers contradict each other.  The tolerances of test_gpu_cache.py hold
unless a test says otherwise."""
import math

import pytest
import torch

from test_gpu_cache import D, U, Case, h  # noqa: F401  (h: the package's fixture)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- factors of a tile
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,length", [(2, 20), (16, 40), (100, 100), (100, 129), (300, 1000)])
def test_zero_queries_and_keys(h, n, length, quantised):
    """All logits are 0: every row is the mean of the values that it sees, however small the powers of two in front of them."""
    c = Case(h, [n], [length], 2, 2, 16, quantised, seed=n)
    c.q = torch.zeros_like(c.q)
    c.k[0] = torch.zeros_like(c.k[0])
    c.fill()
    for causal in (True, False):
        out, lse = c.check(causal)
        assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n", [2, 100])
@pytest.mark.parametrize("scale", [1e-12, 1e-30, 1e-38])
def test_scales_next_to_nothing(h, n, scale, quantised):
    c = Case(h, [n], [n + 37], 2, 2, 16, quantised, seed=n)
    c.q[0] = 0
    c.fill().check(True, softmax_scale=scale)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,length,heads", [(10, 129, 4), (100, 129, 2), (130, 257, 2), (40, 130, 2), (300, 385, 4)])
def test_hidden_nan_keys_alone_in_a_tile(h, n, length, heads, quantised):
    """The keys of the last tile are NaN and only the last tokens may see them."""
    c = Case(h, [n], [length], heads, 2, 16, quantised, seed=n)
    first = (length - 1) // 128 * 128
    c.k[0][first:, :, 0] = math.nan
    c.fill()
    out, lse = h.cache_attn(c.q.cuda(), c.cache, c.batch, return_lse=True)
    sees = torch.arange(length - n, length, device="cuda") >= first  # rows for which everything is NaN
    assert torch.isnan(out[sees].float()).all() and torch.isnan(lse[:, sees]).all()
    c.k[0][first:, :, 0] = 0  # hidden from the others: any number will do
    ro, rl, tol, ltol = c.reference(True)
    c.compare(out[~sees], lse[:, ~sees], ro[~sees], rl[:, ~sees], tol[~sees], ltol[:, ~sees])


# ---------------------------------------------------------------------------------------------- one large key
def by_key(c, causal, rows, scale=D ** -0.5):
    """(out, tolerance) of the given rows of a cache of one sequence, where an error of a logit goes by ITS key, not by the
    row's largest one: with ds_j = scale (sum_d |q_d k_jd|) 128 2^-23 it moves the result by at most
    sum_j softmax_j 2 (ds_j + 2^-20) (|v_j| + |o|)."""
    group, n, length = c.heads // c.kv_heads, c.n[0], c.lengths_l[0]
    k, v = (t.cuda().repeat_interleave(group, 1).transpose(0, 1) for t in c.stored(0))
    x = c.q.cuda().double().transpose(0, 1)
    s = (x @ k.transpose(1, 2)) * scale
    if causal:
        seen = torch.arange(length, device="cuda")[None] <= (length - n + torch.arange(n, device="cuda"))[:, None]
        s = s.masked_fill(~seen, -math.inf)
    w = torch.softmax(s, -1)
    ds = scale * (x.abs() @ k.abs().transpose(1, 2)) * 128 * 2.0 ** -23
    o, a = w @ v, w @ v.abs()
    moved = 2 * (ds + 2.0 ** -20) * w
    tol = U * o.abs() + U * a + moved @ v.abs() + moved.sum(-1, keepdim=True) * o.abs() + (2.0 ** -23 * v.abs().sum(1, keepdim=True) if c.quantised else 0)
    return o.transpose(0, 1)[rows], tol.transpose(0, 1)[rows]


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("power", [10, 18, 24, 30, 60, 110])
@pytest.mark.parametrize("n,length", [(3, 200), (100, 300), (300, 900)])
def test_one_large_key_that_counts_for_nothing(h, n, length, power, quantised):
    """A key 2^power times as large as its neighbours, to which every query is opposed."""
    c = Case(h, [n], [length], 4, 2, 16, quantised, seed=power)
    c.q[..., 0] = c.q[..., 0].abs() + 1
    for j in (5, length - n - 3):
        c.k[0][j] = 0
        c.k[0][j, :, 0] = -(2.0 ** power)
    c.fill()
    for causal in (True, False):
        out = h.cache_attn(c.q.cuda(), c.cache, c.batch, causal=causal)
        ro, tol = by_key(c, causal, slice(None))
        over = (out.double() - ro).abs() - tol
        assert float(over.max()) <= 0, float(over.max())


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("power", [10, 18, 24, 30, 60, 110])
@pytest.mark.parametrize("n,length", [(3, 200), (100, 300), (129, 900)])
def test_hidden_large_keys(h, n, length, power, quantised):
    """The last key is 2^power times as large as the others: nothing of it reaches the rows that do not see it."""
    c = Case(h, [n], [length], 4, 2, 16, quantised, seed=power)
    c.k[0][-1] = (c.k[0][-1].double() * 2.0 ** power).bfloat16()
    c.fill()
    out = h.cache_attn(c.q.cuda(), c.cache, c.batch)
    ro, tol = by_key(c, True, slice(0, n - 1))
    over = (out[: n - 1].double() - ro).abs() - tol
    assert float(over.max()) <= 0, float(over.max())


# ---------------------------------------------------------------------------------------------- sizes of V
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("power", [6, 8, 13, 30, 39, 47, 90])
@pytest.mark.parametrize("n,length", [(4, 640), (1000, 640)])
def test_values_that_grow_along_the_sequence(h, n, length, power, quantised):
    """V of the later keys is 2^power times as large as that of the first ones: pieces whose first tile has small values only."""
    c = Case(h, [n], [length], 40, 40, 32, quantised, seed=power)
    c.v[0][128:] = (c.v[0][128:].double() * 2.0 ** power).bfloat16()
    c.fill()
    for causal in (True, False):
        c.check(causal)


@pytest.mark.parametrize("quantised,power", [(False, 20), (False, 80), (False, 112), (True, 80), (True, 112)])
@pytest.mark.parametrize("n,length,nats", [(4, 640, 40), (1000, 640, 5), (1000, 640, 9), (1000, 640, 40), (300, 2000, 40)])
def test_large_values_under_growing_logits(h, n, length, nats, quantised, power):
    """Keys behind the first tile have logits far above the first ones', and V is so large that unnormalised sums of it
    would leave fp32 if the terms could grow freely.  (The results themselves are far inside it.)"""
    c = Case(h, [n], [length], 40, 40, 32, quantised, seed=nats, v_scale=2.0 ** power)
    c.q[..., 0] = 8
    for j in range(150, length, 90):
        c.k[0][j] = 0
        c.k[0][j, :, 0] = nats / 8 * math.sqrt(D)
    c.fill()
    for causal in (True, False):
        out, _ = c.check(causal)
        assert torch.isfinite(out.float()).all()


# ---------------------------------------------------------------------------------------------- batches that are wrong
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("starts,lengths", [
    ([0, 10, 5, 20], [40, 40, 40]), ([20, 10, 5, 0], [40, 40, 40]), ([0, 0, 0, 21], [40, 40, 40]), ([-1, 4, 5, 20], [40, 40, 40]),
    ([0, 20, 20, 20], [40, -1, 40]), ([0, 20, 20, 20], [40, 40, 1000]), ([0, 7, 7, 3], [40, 40, 40]), ([20, 20, 20, 0], [40, 40, 40])])
def test_every_sequence_of_a_batch_is_checked(h, starts, lengths, quantised):
    """Offsets that decrease or leave the rows and lengths outside the pages are reported by every call, also those of
    sequences that no row is looked up in."""
    from pika_h3_flex_b200 import _lib

    c = Case(h, [8, 4, 8], [40, 40, 40], 2, 2, 16, quantised).fill()
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = h.CacheBatch(c.batch.pages, dev(lengths), dev(starts))
    kv = torch.zeros(20, 2, D, dtype=torch.bfloat16, device="cuda")
    for call in (lambda s: h.cache_write(c.cache, batch, kv, kv, status_word=s),
                 lambda s: h.cache_read(c.cache, batch, 20, status_word=s),
                 lambda s: h.cache_attn(c.q.cuda(), c.cache, batch, status_word=s)):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        call(status)
        with pytest.raises(_lib.H3AError) as e:
            h.check_status(status)
        assert e.value.status == _lib.H3A_ERR_INDEX


def test_an_empty_sequence_among_many_is_checked(h):
    """More sequences than a block has threads; the one that is wrong is far from the rows."""
    from pika_h3_flex_b200 import _lib

    B = 700
    cache = h.KVCache.empty(4, 16, 2)
    starts = torch.zeros(B + 1, dtype=torch.int32)
    starts[1:] = 5
    lengths = torch.full((B,), 5, dtype=torch.int32)
    lengths[650] = 17
    batch = h.CacheBatch(torch.zeros(B, 1, dtype=torch.int32).cuda(), lengths.cuda(), starts.cuda())
    kv = torch.zeros(5, 2, D, dtype=torch.bfloat16, device="cuda")
    for call in (lambda s: h.cache_write(cache, batch, kv, kv, status_word=s), lambda s: h.cache_read(cache, batch, 5, status_word=s),
                 lambda s: h.cache_attn(kv, cache, batch, status_word=s)):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        call(status)
        with pytest.raises(_lib.H3AError) as e:
            h.check_status(status)
        assert e.value.status == _lib.H3A_ERR_INDEX


def test_expanded_exponents_are_read_but_not_written(h):
    from pika_h3_flex_b200 import _lib

    c = Case(h, [20], [20], 2, 2, 16, True)
    codes = torch.randn(c.cache.k.shape, device="cuda").to(torch.float8_e4m3fn)
    one = torch.full((1, 1, 1), 124, dtype=torch.uint8, device="cuda").expand(c.cache.k.shape[:3])
    cache = h.KVCache(codes, codes, one, one)
    kv = torch.zeros(20, 2, D, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(_lib.H3AError) as e:
        h.cache_write(cache, c.batch, kv, kv)
    assert e.value.status == _lib.H3A_ERR_ALIGN
    got, _ = h.cache_read(cache, c.batch, 20)
    rows = codes[c.batch.pages[0].long()].reshape(-1, 2, D)[:20]
    assert torch.equal(got.double(), rows.double() / 8)


# ---------------------------------------------------------------------------------------------- a caller's workspace
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("fill", [0, 1, 127, 255])
def test_what_a_workspace_held_before_does_not_matter(h, fill, quantised):
    """One workspace for calls of several shapes, one after the other, each on what the one before left in it: descriptions of
    items in parts and partial results of other shares."""
    shapes = [([300, 40, 1], [900, 2000, 500], 6, 2), ([150], [1100], 4, 4), ([2, 1], [3000, 700], 8, 2), ([1], [40000], 8, 1), ([700], [700], 2, 2)]
    cases = [Case(h, *s, 32, quantised, seed=i).fill() for i, s in enumerate(shapes)]
    want = [h.cache_attn(c.q.cuda(), c.cache, c.batch, return_lse=True) for c in cases]
    need = max(h.cache_attn_workspace_bytes(c.cache, c.batch, c.rows, c.heads) for c in cases)
    workspace = torch.full((need,), fill, dtype=torch.uint8, device="cuda")
    for _ in range(20):
        for c, (out, lse) in zip(cases, want):
            got = h.cache_attn(c.q.cuda(), c.cache, c.batch, return_lse=True, workspace=workspace)
            assert torch.equal(got[0], out) and torch.equal(got[1], lse)


def test_a_workspace_must_be_contiguous(h):
    c = Case(h, [2], [20], 4, 2, 16, False).fill()
    need = h.cache_attn_workspace_bytes(c.cache, c.batch, 2, 4)
    for w in (torch.empty(32, dtype=torch.uint8, device="cuda")[:1].expand(need), torch.empty(need, 2, dtype=torch.uint8, device="cuda")[:, 0]):
        with pytest.raises(ValueError, match="contiguous"):
            h.cache_attn(c.q.cuda(), c.cache, c.batch, workspace=w)


# ---------------------------------------------------------------------------------------------- values that are not finite
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,length,heads,kv_heads", [([700], [900], 4, 4), ([300, 20, 400], [2000, 20, 500], 6, 2), ([257], [400], 2, 1), ([150], [150], 128, 1)])
def test_values_that_are_not_finite_all_over(h, n, length, heads, kv_heads, quantised):
    """NaN and infinities in V of many tokens, every item's first and last visible keys among them: each reaches the rows
    that see it, in its own dimension (a quantised row: in all), and no other row, also in items of later sequences."""
    c = Case(h, n, length, heads, kv_heads, 16, quantised, seed=len(n))
    for b, (m, x) in enumerate(zip(n, length)):
        for j in range(x - m, x, 37):
            c.v[b][j, :, j % D] = (math.nan, math.inf, -math.inf)[j % 3]
            c.v[b][j, 0, 5] = math.inf
    c.fill()
    for causal in (True, False):
        out, lse = h.cache_attn(c.q.cuda(), c.cache, c.batch, causal=causal, return_lse=True)
        c.compare(out, lse, *c.reference(causal))


# ---------------------------------------------------------------------------------------------- waits that run out
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("limit_ns", [1, 2048, 4096, 8192, 16384, 65536])
def test_a_wait_that_runs_out_is_reported(h, limit_ns, quantised):
    """A limit shorter than what a wait takes: the call returns, with the timeout in the status word or with right results, and
    the device is as good as before."""
    from pika_h3_flex_b200 import _lib

    c = Case(h, [500, 1, 90], [3000, 700, 90], 8, 4, 32, quantised, seed=3).fill()
    q = c.q.cuda()
    want = h.cache_attn(q, c.cache, c.batch, return_lse=True)
    for _ in range(3):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out, lse = h.cache_attn(q, c.cache, c.batch, return_lse=True, status_word=status, wait_limit_ns=limit_ns)
        try:
            h.check_status(status)
        except _lib.H3AError as e:
            assert e.status == _lib.H3A_ERR_TIMEOUT
            assert 33 <= int(status.item()) & 0xFF <= 49
        else:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        status.zero_()
        out, lse = h.cache_attn(q, c.cache, c.batch, return_lse=True, status_word=status)
        assert h.read_status(status) == 0 and torch.equal(out, want[0]) and torch.equal(lse, want[1])


# ---------------------------------------------------------------------------------------------- precision
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,length,heads,kv_heads", [([1], [700], 8, 2), ([1, 2, 1], [50, 3000, 129], 10, 2), ([5], [500], 2, 2), ([4], [2000], 4, 1), ([1], [30000], 8, 1)])
def test_few_rows_keep_their_probabilities(h, n, length, heads, kv_heads, quantised):
    """Up to 16 query rows per K/V head: probabilities lose at most 2^-16 of themselves (bf16, in two parts) or 2^-11 (fp16, one
    part), so that with ds and r of test_gpu_cache.py a result is off by u |o| + (that + 2 (ds + r)) A, and by what fp16's last
    place takes."""
    c = Case(h, n, length, heads, kv_heads, 32, quantised, seed=9).fill()
    for causal in (True, False):
        out, lse = h.cache_attn(c.q.cuda(), c.cache, c.batch, causal=causal, return_lse=True)
        ro, rl, tol, ltol = c.reference(causal)
        a = torch.zeros_like(ro)  # sum_j softmax_j |v_j|
        for b, (m, x) in enumerate(zip(n, length)):
            k, v = (t.cuda().repeat_interleave(heads // kv_heads, 1).transpose(0, 1) for t in c.stored(b))
            s = c.q[c.starts[b] : c.starts[b] + m].cuda().double().transpose(0, 1) @ k.transpose(1, 2) * D ** -0.5
            if causal:
                s = s.masked_fill(torch.arange(x, device="cuda")[None] > (x - m + torch.arange(m, device="cuda"))[:, None], -math.inf)
            a[c.starts[b] : c.starts[b] + m] = (torch.softmax(s, -1) @ v.abs()).transpose(0, 1)
        c.compare(out, lse, ro, rl, tol - (U - (2.0 ** -11 if quantised else 2.0 ** -16)) * a, ltol)


# ---------------------------------------------------------------------------------------------- logits without bounds
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("power", [10, 28, 40, 90, 115])
@pytest.mark.parametrize("n,length,j", [(1, 127, 3), (3, 700, 600), (100, 300, 5), (100, 300, 190), (300, 900, 599), (40, 40, 0)])
def test_logits_of_any_size(h, n, length, j, power, quantised):
    """Logits that differ by far more than fp32 resolves at their size: a row is the value of its one key, exactly."""
    c = Case(h, [n], [length], 4, 2, 16, quantised, seed=power)
    c.q[..., 0] = c.q[..., 0].abs() + 1
    v = c.stored(0)[1][j].repeat_interleave(2, 0).cuda()  # [heads, 128]
    for sign in (1, -1):
        if sign > 0:  # one key far above the others
            c.k[0][j] = 0
            c.k[0][j, :, 0] = 2.0 ** power
        else:  # all far below zero, one the least
            c.k[0][:] = 0
            c.k[0][:, :, 0] = -(2.0 ** (power + 1))
            c.k[0][j, :, 0] = -(2.0 ** power)
        c.fill()
        for causal in (True, False):
            out, lse = h.cache_attn(c.q.cuda(), c.cache, c.batch, causal=causal, return_lse=True)
            sees = torch.arange(length - n, length, device="cuda") >= (j if causal else 0)
            logit = sign * c.q[..., 0].cuda().double() * 2.0 ** power * D ** -0.5  # above the next one by its own size or so
            assert torch.isfinite(out.float()).all() and torch.isfinite(lse).all()
            if power > 10:
                assert torch.equal(out[sees].double(), v.expand(n, 4, D)[sees])
                assert ((lse.T[sees].double() - logit[sees]).abs() <= 2.0 ** -18 * logit[sees].abs()).all()
