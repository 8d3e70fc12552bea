"""GPU: the paged K/V cache (cache_write, cache_read, cache_attn) against plain implementations in 64 bits.

Write and read are exact: e4m3 rounding and the power-of-two exponent are restated below in 64-bit arithmetic, and what is
read back is a bf16 number.  Attention tolerance, element by element, with u = 2^-8 (half a bf16 step, relative):
  u |o|          the rounding of the result,
  u A            the rounding of each probability before P V, where A = sum_j softmax_j |v_j|,
  2 (ds + r) A   errors of the logits and of the exponentials: ds = scale (max_j sum_d |q_d k_jd|) 128 2^-23 (fp32 sums of 128
                 exact products, truncating adders allowed for), r = 2^-20 (exponential, scaling, 8-bit lazy rescale, sums),
and for a quantised cache, whose probabilities are fp16 numbers with a last place of 2^-24, so that terms far below the row's
largest vanish however large the relative error of one that stands alone would be: at most half of that place a term, against
a largest term of at least 2^2 (many rows) or 2^6 (few rows; each relative to V's unit, which is at most 2^8 above the row's
own), divided by a sum that is at least the largest term:
  2^-25 2^-2 S  or  2^-25 2^-6 2^8 S,  S = sum_j |v_j| over the keys the row sees,
and for the log-sum-exp ds + (keys) 2^-24 + 2^-21 (1 + |lse| + max logit)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
D = 128


@pytest.fixture(scope="module")
def h(lib):
    import pika_h3_flex_b200 as pkg

    assert torch.cuda.is_available()
    return pkg


# ---------------------------------------------------------------------------------------------- plain forms
def pow2(k):
    return torch.ldexp(torch.ones(k.shape, dtype=torch.float64, device=k.device), k.to(torch.int64))


def quantise(x):
    """Rows of bf16 values as (codes, exponent bytes), both in plain numbers; rows with NaN or infinity: byte 255."""
    x = x.double()
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    top = torch.where(bad, torch.ones_like(top), top)
    m, e = torch.frexp(torch.where(top == 0, torch.ones_like(top), top))
    k = torch.where(m <= 0.875, e - 9, e - 8)  # 448 = 0.875 * 2^9
    k = torch.where(top == 0, torch.full_like(k, -120), k).clamp(min=-120)
    y = x / pow2(k)[..., None]
    _, ey = torch.frexp(y.abs().clamp(min=2.0 ** -6))
    step = pow2(ey - 4)  # 4 significant bits, no finer than 2^-9
    c = torch.round(y / step) * step
    c = torch.where((k == 120)[..., None], c.clamp(-240, 240), c)  # 256 * 2^120 is no bf16 number
    return c, torch.where(bad, torch.full_like(k, 255), k + 127)


def values(c, e):
    x = c * pow2(e - 127)[..., None]
    return torch.where((e == 255)[..., None], torch.full_like(x, math.nan), x)


class Case:
    """A cache with sequences in scattered pages, and the 64-bit values of every token."""

    def __init__(self, h, n, lengths, heads, kv_heads, page, quantised, seed=0, layout="head", spare=2, v_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.h, self.n, self.lengths_l, self.page, self.quantised = h, n, lengths, page, quantised
        self.heads, self.kv_heads = heads, kv_heads
        per = [-(-x // page) for x in lengths]
        n_pages = sum(per) + spare
        order = torch.randperm(n_pages, generator=g).tolist()
        self.pages = torch.full((len(n), max(max(per), 1)), -1, dtype=torch.int32)  # unused entries name no page
        self.seq_pages = []
        for b, x in enumerate(per):
            ids = [order.pop() for _ in range(x)]
            self.seq_pages.append(ids)
            self.pages[b, :x] = torch.tensor(ids, dtype=torch.int32)
        self.unused = order
        self.starts = [0]
        for x in n:
            self.starts.append(self.starts[-1] + x)
        self.rows = self.starts[-1]
        self.k = [torch.randn(x, kv_heads, D, generator=g).bfloat16() for x in lengths]
        self.v = [(v_scale * torch.randn(x, kv_heads, D, generator=g)).bfloat16() for x in lengths]
        self.q = torch.randn(max(self.rows, 1), heads, D, generator=g).bfloat16()[: self.rows]
        self.cache = self.make_cache(layout, n_pages)
        self.batch = h.CacheBatch(self.pages.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                                  torch.tensor(self.starts, dtype=torch.int32, device="cuda"))

    def make_cache(self, layout, n_pages):
        h, p, hk = self.h, self.page, self.kv_heads
        if layout == "head":
            c = h.KVCache.empty(n_pages, p, hk, self.quantised)
        else:  # token-major pages inside one tensor that holds K and V side by side, with room between the rows
            dt = torch.float8_e4m3fn if self.quantised else torch.bfloat16
            both = torch.empty(n_pages, p, 2, hk + 1, D + 16, dtype=dt, device="cuda")
            ex = torch.empty(n_pages, p, 2, hk, dtype=torch.uint8, device="cuda") if self.quantised else None
            c = h.KVCache(both[:, :, 0, :hk, :D], both[:, :, 1, :hk, :D], *((ex[:, :, 0], ex[:, :, 1]) if self.quantised else (None, None)))
        # nothing in a fresh cache may matter: NaN everywhere (all-ones bytes), exponent bytes 255
        for t in (c.k, c.v):
            t.view(torch.uint8).fill_(255) if self.quantised else t.fill_(math.nan)
        if self.quantised:
            c.k_exp.fill_(255)
            c.v_exp.fill_(255)
        return c

    def fill(self):
        """All tokens enter the cache through one write of whole sequences."""
        keep = [b for b, x in enumerate(self.lengths_l) if x]
        if not keep:
            return self
        lens = [self.lengths_l[b] for b in keep]
        st = [0]
        for x in lens:
            st.append(st[-1] + x)
        batch = self.h.CacheBatch(self.pages[keep].cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.tensor(st, dtype=torch.int32, device="cuda"))
        self.h.cache_write(self.cache, batch, torch.cat([self.k[b] for b in keep]).cuda(), torch.cat([self.v[b] for b in keep]).cuda())
        return self

    def stored(self, b):
        k, v = self.k[b], self.v[b]
        if self.quantised:
            return values(*quantise(k)), values(*quantise(v))
        return k.double(), v.double()

    def reference(self, causal, scale=D ** -0.5, q=None, max_new=None):
        """(out, lse, tolerance of out, tolerance of lse) in 64 bits, on the GPU."""
        dev, group = "cuda", self.heads // self.kv_heads
        q = (self.q if q is None else q).to(dev).double()
        few = (max_new or -(-self.rows // len(self.n))) * group <= 16  # which kernel runs
        absolute = (2.0 ** -23 if few else 2.0 ** -27) if self.quantised else 0.0
        out = torch.zeros(self.rows, self.heads, D, dtype=torch.float64, device=dev)
        tol = torch.zeros_like(out)
        lse = torch.full((self.heads, self.rows), -math.inf, dtype=torch.float64, device=dev)
        ltol = torch.zeros_like(lse)
        for b, (n, length) in enumerate(zip(self.n, self.lengths_l)):
            if n == 0 or length == 0:
                continue
            k, v = (t.to(dev).repeat_interleave(group, 1).transpose(0, 1) for t in self.stored(b))  # [H, len, D]
            x = q[self.starts[b] : self.starts[b] + n].transpose(0, 1)
            s = (x @ k.transpose(1, 2)) * scale
            seen = torch.ones(n, length, dtype=torch.bool, device=dev)
            if causal:
                seen = torch.arange(length, device=dev)[None] <= (length - n + torch.arange(n, device=dev))[:, None]
            s = s.masked_fill(~seen, -math.inf)
            ds = scale * (x.abs() @ k.abs().transpose(1, 2)).masked_fill(~seen, 0).nan_to_num().amax(-1) * 128 * 2.0 ** -23
            m = s.amax(-1)
            m0 = torch.where(m == -math.inf, torch.zeros_like(m), m)
            p = torch.exp(s - m0[..., None])
            p = torch.where(seen, p, torch.zeros_like(p))
            l = p.sum(-1)
            w = p / torch.where(l == 0, torch.ones_like(l), l)[..., None]
            vz = v.nan_to_num(0, 0, 0)
            o = w @ vz
            poison = torch.zeros_like(o)  # values that are not finite, for the rows that see them
            odd = torch.nonzero(~torch.isfinite(v).all(-1).all(0)).flatten().tolist()
            for j in odd:
                poison += torch.where(seen[:, j][None, :, None] & ~torch.isfinite(v[:, j])[:, None], v[:, j][:, None], torch.zeros_like(o))
            o = o + poison
            a = w @ vz.abs()
            r = slice(self.starts[b], self.starts[b] + n)
            out[r] = o.transpose(0, 1)
            tol[r] = (U * o.abs() + (U + 2 * (ds + 2.0 ** -20))[..., None] * a + absolute * (seen.double() @ vz.abs())).transpose(0, 1)
            lse[:, r] = torch.where(l == 0, torch.full_like(l, -math.inf), l.log() + m0)
            ltol[:, r] = ds + length * 2.0 ** -24 + 2.0 ** -21 * (1 + m0.abs() + (l.clamp(min=1e-300).log() + m0).abs())
        return out, lse, tol, ltol

    def check(self, causal, **kw):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out, lse = self.h.cache_attn(self.q.cuda(), self.cache, self.batch, causal=causal, return_lse=True, status_word=status, **kw)
        assert self.h.read_status(status) == 0
        self.compare(out, lse, *self.reference(causal, kw.get("softmax_scale", 0) or D ** -0.5, max_new=kw.get("max_new")))
        return out, lse

    @staticmethod
    def compare(out, lse, ro, rl, tol, ltol):
        out, lse = out.double(), lse.double()
        fine = torch.isfinite(ro)
        assert torch.equal(torch.isnan(out), torch.isnan(ro)) and torch.equal(out[~fine & ~torch.isnan(ro)], ro[~fine & ~torch.isnan(ro)])
        over = ((out - ro).abs() - tol)[fine]
        assert over.numel() == 0 or float(over.max()) <= 0, float(over.max())
        fin = torch.isfinite(rl)
        assert torch.equal(lse[~fin & ~torch.isnan(rl)], rl[~fin & ~torch.isnan(rl)])
        lo = ((lse - rl).abs() - ltol)[fin]
        assert lo.numel() == 0 or float(lo.max()) <= 0, float(lo.max())


# ---------------------------------------------------------------------------------------------- write and read
def wide_rows(rows, heads, g):
    """Rows over the whole range of the type: ordinary ones, tiny and huge ones, zeros, the largest number, subnormals."""
    x = torch.randn(rows, heads, D, generator=g, dtype=torch.float64)
    x = x * pow2(torch.randint(-125, 120, (rows, heads), generator=g))[..., None]
    x[::7] = torch.randn(x[::7].shape, generator=g, dtype=torch.float64)
    x = x.bfloat16()
    flat = x.view(-1, D)
    flat[3::11] = 0
    flat[5::13, 2] = torch.finfo(torch.bfloat16).max
    flat[6::17] = torch.tensor(2.0 ** -133, dtype=torch.float64).bfloat16()
    return x


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,lengths,kv_heads,page,layout", [
    ([1], [1], 1, 16, "head"), ([0, 1, 7], [5, 33, 7], 3, 16, "token"), ([200, 1, 130], [333, 48, 130], 5, 48, "head"),
    ([64] * 9, [64 + 16 * i for i in range(9)], 2, 256, "token"), ([1000], [1000], 40, 128, "head")])
def test_write_and_read_are_exact(h, quantised, n, lengths, kv_heads, page, layout):
    g = torch.Generator().manual_seed(5)
    c = Case(h, n, lengths, kv_heads, kv_heads, page, quantised, layout=layout)
    k, v = wide_rows(c.rows, kv_heads, g), wide_rows(c.rows, kv_heads, g)
    before = [t.view(torch.uint8).clone() for t in (c.cache.k, c.cache.v)]
    big = torch.empty(c.rows, 2, kv_heads, D, dtype=torch.bfloat16, device="cuda")  # K and V rows interleaved
    big[:, 0], big[:, 1] = k.cuda(), v.cuda()
    h.cache_write(c.cache, c.batch, big[:, 0], big[:, 1])
    out = tuple(torch.full((c.rows + 3, kv_heads, D), 9.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    h.cache_read(c.cache, c.batch, out=out)
    for x, y, pool, old in ((k, out[0], c.cache.k, before[0]), (v, out[1], c.cache.v, before[1])):
        want = values(*quantise(x)) if quantised else x.double()
        assert torch.equal(y[: c.rows].cpu().double(), want)
        assert (y[c.rows :] == 9).all()  # rows behind the last sequence
        # and nothing else in the pool moved
        touched = torch.zeros(pool.shape[:2], dtype=torch.bool)
        for b, (m, length) in enumerate(zip(n, lengths)):
            for p in range(length - m, length):
                touched[c.pages[b, p // page], p % page] = True
        same = (pool.view(torch.uint8) == old).flatten(2).all(-1).cpu()
        assert same[~touched].all()
    if quantised:  # the bytes themselves
        b, p = len(n) - 1, lengths[-1] - 1
        code, e = quantise(k[-1])
        at = (int(c.pages[b, p // page]), p % page)
        assert torch.equal(c.cache.k_exp[at].cpu().long(), e)
        assert torch.equal(c.cache.k[at].float().cpu().double(), code)


def test_rows_that_are_not_finite(h):
    c = Case(h, [4], [4], 2, 2, 16, True)
    k = torch.randn(4, 2, D).bfloat16()
    k[0, 0, 5], k[1, 1, 7], k[2, 0, 0] = math.nan, math.inf, -math.inf
    h.cache_write(c.cache, c.batch, k.cuda(), k.cuda())
    got, _ = h.cache_read(c.cache, c.batch, 4)
    got = got.cpu()
    for r, x in ((0, 0), (1, 1), (2, 0)):
        assert torch.isnan(got[r, x]).all()
    ok = torch.isfinite(k).all(-1)
    assert torch.equal(got[ok].double(), values(*quantise(k))[ok])
    c = Case(h, [4], [4], 2, 2, 16, False)
    h.cache_write(c.cache, c.batch, k.cuda(), k.cuda())
    got, _ = h.cache_read(c.cache, c.batch, 4)
    assert torch.equal(got.view(torch.int16).cpu(), k.view(torch.int16))


def test_positions_before_the_cache(h):
    """More new rows than the sequence holds: the first ones have no position."""
    c = Case(h, [5], [3], 2, 2, 16, False)
    k, v = torch.randn(5, 2, D).bfloat16(), torch.randn(5, 2, D).bfloat16()
    h.cache_write(c.cache, c.batch, k.cuda(), v.cuda())
    gk, gv = (t.cpu() for t in h.cache_read(c.cache, c.batch, 5))
    assert (gk[:2] == 0).all() and (gv[:2] == 0).all()
    assert torch.equal(gk[2:], k[2:]) and torch.equal(gv[2:], v[2:])
    c.k[0], c.v[0] = k[2:], v[2:]
    out, lse = c.check(True)
    assert (out[:2] == 0).all() and (lse[:, :2] == -math.inf).all()
    c.check(False)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,length", [(200, 150), (400, 20), (129, 0)])
def test_more_rows_than_keys(h, n, length, quantised):
    c = Case(h, [n, 30], [length, 40], 2, 2, 16, quantised, seed=n).fill()
    out, lse = c.check(True)
    assert (out[: n - length] == 0).all() and (lse[:, : n - length] == -math.inf).all()
    c.check(False)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("max_new", [None, 1, 400])
def test_tokens_and_a_chunk_in_one_batch(h, max_new, quantised):
    """Either kernel computes any batch; the longest sequence's rows only choose which."""
    Case(h, [1] * 20 + [400] + [1] * 40, [100 + 30 * b for b in range(61)], 8, 4, 32, quantised, seed=5).fill().check(True, max_new=max_new)


# ---------------------------------------------------------------------------------------------- attention
SHAPES = [
    # new rows, lengths, heads, K/V heads, page
    ([1], [1], 1, 1, 16),
    ([1], [16], 4, 2, 16),
    ([1, 1, 1], [15, 17, 129], 8, 8, 16),
    ([1] * 7, [0, 1, 127, 128, 129, 1000, 4097], 20, 4, 48),
    ([2, 3, 1, 0, 4], [2, 90, 1, 40, 300], 15, 3, 32),
    ([1, 1], [3000, 20000], 40, 8, 128),
    ([1], [70000], 6, 2, 64),
    ([5], [500], 64, 2, 256),
    ([1] * 40, [37 * i for i in range(40)], 7, 1, 16),
    ([17], [17], 3, 3, 16),
    ([128], [128], 2, 2, 16),
    ([129], [1000], 2, 2, 112),
    ([300, 1, 77, 0, 256], [300, 900, 78, 10, 2000], 6, 2, 48),
    ([257], [515], 5, 1, 64),
    ([40], [9000], 21, 3, 80),
    ([700], [1500], 8, 8, 128),
    ([3], [200], 256, 2, 16),
]


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,lengths,heads,kv_heads,page", SHAPES)
def test_attention(h, n, lengths, heads, kv_heads, page, causal, quantised):
    Case(h, n, lengths, heads, kv_heads, page, quantised, seed=len(n) + lengths[-1]).fill().check(causal)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,lengths", [([2, 1], [50, 700]), ([150], [1100])])
def test_attention_in_other_layouts(h, n, lengths, quantised):
    """Token-major pages with gaps, queries and outputs as views of wider tensors, a scale of its own."""
    c = Case(h, n, lengths, 10, 2, 32, quantised, seed=3, layout="token").fill()
    wide = torch.zeros(10, c.rows, 3 * D, dtype=torch.bfloat16, device="cuda")
    q = wide[:, :, D : 2 * D].transpose(0, 1)
    q.copy_(c.q)
    room = torch.full((c.rows + 2, 12, D), 5.0, dtype=torch.bfloat16, device="cuda")
    out, lse = h.cache_attn(q, c.cache, c.batch, softmax_scale=0.2, out=room[: c.rows, 1:11], return_lse=True)
    c.compare(out, lse, *c.reference(True, 0.2))
    assert (room[c.rows :] == 5).all() and (room[:, 0] == 5).all() and (room[:, 11] == 5).all()


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n", [1, 170])
def test_rows_at_odd_multiples_of_16_bytes(h, n, quantised):
    c = Case(h, [n], [n + 300], 4, 2, 16, quantised, seed=5).fill()
    room = torch.full((n * 4 * D + 8,), 5.0, dtype=torch.bfloat16, device="cuda")
    q = torch.empty(n * 4 * D + 8, dtype=torch.bfloat16, device="cuda")[8:].view(n, 4, D)
    q.copy_(c.q)
    out, lse = h.cache_attn(q, c.cache, c.batch, out=room[8:].view(n, 4, D), return_lse=True)
    c.compare(out, lse, *c.reference(True))
    assert (room[:8] == 5).all()


# Few items in very many parts: every share of the device has one of the same few rows.
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,lengths,heads,kv_heads", [([1], [70000], 8, 1), ([2], [40001], 5, 1), ([1, 1], [30003, 17], 2, 2), ([0, 3, 0], [5, 9000, 800], 4, 2), ([7], [300], 2, 1)])
def test_few_rows_over_long_contexts(h, n, lengths, heads, kv_heads, quantised):
    c = Case(h, n, lengths, heads, kv_heads, 64, quantised, seed=8).fill()
    for causal in (True, False):
        out, lse = h.cache_attn(c.q.cuda(), c.cache, c.batch, causal=causal, return_lse=True)
        c.compare(out, lse, *c.reference(causal))


# Enough rows that a half-warp takes whole tokens, whose exponents leave together: more heads than meet at a time, and few.
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,lengths,kv_heads,page,layout", [([700, 601], [700, 640], 130, 16, "head"), ([1300, 0, 77], [1300, 9, 100], 3, 32, "token")])
def test_many_rows_are_exact(h, quantised, n, lengths, kv_heads, page, layout):
    test_write_and_read_are_exact(h, quantised, n, lengths, kv_heads, page, layout)


# Items of one key tile, of none at all (rows before the sequence) and of many, on few enough heads that shares end within
# an item's set-up as well as between its tiles; results must not depend on where the cuts are.
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("heads", [1, 3, 7])
def test_shares_that_end_anywhere(h, heads, quantised):
    n, lengths = [300, 700, 40, 257, 1, 900], [20, 90, 129, 3000, 1000, 128]
    c = Case(h, n, lengths, heads, heads, 16, quantised, seed=6).fill()
    for causal in (True, False):
        out, lse = h.cache_attn(c.q.cuda(), c.cache, c.batch, causal=causal, return_lse=True)
        c.compare(out, lse, *c.reference(causal))


@pytest.mark.parametrize("n", [1, 6, 140])
def test_rows_outside_every_sequence_are_left_alone(h, n):
    c = Case(h, [n], [400], 4, 4, 16, False).fill()
    q = torch.randn(n + 9, 4, D, dtype=torch.bfloat16, device="cuda")
    q[4 : 4 + n] = c.q.cuda()
    batch = h.CacheBatch(c.batch.pages, c.batch.lengths, torch.tensor([4, 4 + n], dtype=torch.int32, device="cuda"))
    out = torch.full((n + 9, 4, D), 3.0, dtype=torch.bfloat16, device="cuda")
    h.cache_attn(q, c.cache, batch, out=out)
    assert (out[:4] == 3).all() and (out[4 + n :] == 3).all()
    ro, _, tol, _ = c.reference(True)
    assert ((out[4 : 4 + n].double() - ro).abs() <= tol).all()


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,length", [(4, 50), (9, 9), (3, 300), (200, 333), (130, 130), (300, 900)])
def test_hidden_values_that_are_not_finite(h, n, length, quantised):
    """NaN and infinities in K and V of tokens that the causal mask hides from some rows reach exactly the rows that see
    them; pages are NaN behind the last key (make_cache)."""
    c = Case(h, [n, 1], [length, 1], 2, 2, 16, quantised, seed=n)
    for j, d, x in ((n - 1, 3, math.nan), (n // 2, 70, math.inf), (n // 2 + 1, 70, -math.inf)):
        c.v[0][length - n + min(j, n - 1), 0, d] = x
    c.k[0][length - 1, 1, 0] = math.nan
    c.fill()
    out, lse = h.cache_attn(c.q.cuda(), c.cache, c.batch, return_lse=True)
    ro, rl, tol, ltol = c.reference(True)
    # a NaN key makes the logit, and so everything of the rows that see it, NaN
    ro[n - 1, 1], rl[1, n - 1] = math.nan, math.nan
    c.compare(out, lse, ro, rl, tol, ltol)
    assert torch.isnan(lse[1, n - 1])
    assert torch.isfinite(out[: n // 2].float()).all()


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,length", [(1, 5000), (2, 200), (64, 3000), (300, 2000)])
def test_large_logits_and_growing_maxima(h, n, length, quantised):
    """Keys whose logits grow along the sequence far past the range of the exponential: every tile moves the maximum."""
    c = Case(h, [n], [length], 2, 1, 16, quantised, seed=n)
    c.k[0] = (c.k[0].float() * torch.linspace(0.1, 30, length)[:, None, None]).bfloat16()
    c.q = (c.q.float() * 4).bfloat16()
    c.fill().check(True)
    c.k[0] = c.k[0].flip(0)
    c.fill().check(False)


@pytest.mark.parametrize("quantised", [False, True])
def test_many_short_pieces_some_done_twice(h, quantised):
    """More pieces per SM than are handed out at a time, of more sequences than a warp looks over, in some of which late
    keys outgrow the first ones."""
    c = Case(h, [20 + b % 5 for b in range(200)], [150 + b for b in range(200)], 32, 32, 16, quantised, seed=1)
    for b in range(0, 200, 7):
        c.k[b][140:] *= 30
    c.fill().check(True)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,length,heads,kv_heads", [(2000, 300, 40, 40), (2100, 129, 40, 8), (9600, 77, 4, 4)])
def test_whole_items_in_rounds(h, n, length, heads, kv_heads, quantised):
    """One sequence without a mask and with more items than SMs: whole items are dealt out, the rest is cut."""
    Case(h, [n], [length], heads, kv_heads, 32, quantised, seed=n).fill().check(False)


def test_quantised_rows_of_very_different_sizes(h):
    """Exponents of K and V rows over many powers of two, beyond what one multiplication can apply."""
    for n in (1, 100):
        c = Case(h, [n], [400], 4, 2, 32, True, seed=n)
        g = torch.Generator().manual_seed(n)
        k = torch.randint(-40, 1, (400, 2), generator=g)
        v = torch.randint(-110, 100, (400, 2), generator=g)
        c.k[0] = (c.k[0].double() * pow2(k)[..., None]).bfloat16()
        c.v[0] = (c.v[0].double() * pow2(v)[..., None]).bfloat16()
        c.fill().check(True)


@pytest.mark.parametrize("n", [1, 150])
def test_far_pages_of_a_large_cache(h, n):
    """Offsets beyond 2^32 bytes and 2^31 elements."""
    pages, page, kv = 35000, 64, 16
    c = Case(h, [n], [300], 16, kv, page, False, spare=0)
    big = h.KVCache.empty(pages, page, kv)  # 9.2 GB each for K and V
    far = torch.tensor([[pages - 1, pages - 2, 3, pages - 7, pages - 3]], dtype=torch.int32, device="cuda")
    c.cache, c.pages = big, far.cpu()
    c.batch = h.CacheBatch(far, c.batch.lengths, c.batch.starts)
    c.fill().check(True)
    k, _ = h.cache_read(big, c.batch, n)
    assert torch.equal(k.cpu(), c.k[0][300 - n :])


@pytest.mark.parametrize("quantised", [False, True])
def test_chunks_and_tokens_as_they_are_used(h, quantised):
    """Three sequences grow by chunks and then token by token; a page table that grows with them; every step equals the
    attention over everything so far, and at the end the cache reads back as what was written."""
    steps = [[130, 1, 40], [1, 260, 7], [1, 1, 1], [1, 0, 1], [3, 1, 2]]
    total = [sum(s[b] for s in steps) for b in range(3)]
    c = Case(h, total, total, 8, 2, 32, quantised, seed=11)
    have = [0, 0, 0]
    for n in steps:
        at = list(have)
        have = [x + y for x, y in zip(have, n)]
        st = [0, n[0], n[0] + n[1], sum(n)]
        batch = h.CacheBatch(c.batch.pages, torch.tensor(have, dtype=torch.int32, device="cuda"), torch.tensor(st, dtype=torch.int32, device="cuda"))
        new = lambda x: torch.cat([x[b][at[b] : have[b]] for b in range(3)]).cuda()  # noqa: E731
        h.cache_write(c.cache, batch, new(c.k), new(c.v))
        q = torch.cat([c.q[c.starts[b] + at[b] : c.starts[b] + have[b]] for b in range(3)])
        out, lse = h.cache_attn(q.cuda(), c.cache, batch, return_lse=True)
        part = Case.__new__(Case)
        part.__dict__.update(c.__dict__)
        part.n, part.lengths_l, part.starts, part.rows, part.q = n, have, st, st[-1], q
        part.k, part.v = [c.k[b][: have[b]] for b in range(3)], [c.v[b][: have[b]] for b in range(3)]
        part.compare(out, lse, *part.reference(True))
    k, v = h.cache_read(c.cache, c.batch, c.rows)
    for b in range(3):
        wk, wv = c.stored(b)
        assert torch.equal(k[c.starts[b] : c.starts[b + 1]].cpu().double(), wk) and torch.equal(v[c.starts[b] : c.starts[b + 1]].cpu().double(), wv)


def test_after_the_preparation_as_one_path(h):
    """qk_prep -> cache_write -> cache_attn over a clip equals the package's dense attention over the same rows."""
    L, H = 700, 4
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(L, H, D, generator=g).bfloat16().cuda() for _ in range(3))
    tab = h.rope_table(h.position_grid((6, 10, 10), 100).cuda())
    qp, kp, _, _ = h.qk_prep(q, k, tab, tab)
    c = Case(h, [L], [L], H, H, 64, False)
    h.cache_write(c.cache, c.batch, kp, v)
    got = h.cache_attn(qp, c.cache, c.batch, causal=False)
    c.q, c.k[0], c.v[0] = qp.cpu(), kp.cpu(), v.cpu()
    ro, _, tol, _ = c.reference(False)
    assert ((got.double() - ro).abs() <= tol).all()
    want = h.attn_fwd(qp, kp, v)
    assert ((got.double() - want.double()).abs() <= 2 * tol).all()


def test_captured_and_replayed(h):
    """A captured write + attention whose lengths and rows change between replays; a second graph alongside."""
    c = Case(h, [1, 1], [600, 40], 8, 2, 16, True, seed=4).fill()
    q, k, v = (torch.zeros(2, x, D, dtype=torch.bfloat16, device="cuda") for x in (8, 2, 2))
    lengths = torch.tensor([1, 1], dtype=torch.int32, device="cuda")
    batch = h.CacheBatch(c.batch.pages, lengths, c.batch.starts)

    def step():
        h.cache_write(c.cache, batch, k, v)
        return h.cache_attn(q, c.cache, batch, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got))
    c.fill()
    for turn, lens in enumerate([[600, 40], [17, 3], [333, 40]]):
        lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        part = Case.__new__(Case)
        part.__dict__.update(c.__dict__)
        part.lengths_l = lens
        part.k, part.v = [c.k[b][: lens[b]] for b in range(2)], [c.v[b][: lens[b]] for b in range(2)]
        q.copy_(c.q)
        k.copy_(torch.stack([c.k[b][lens[b] - 1] for b in range(2)]))
        v.copy_(torch.stack([c.v[b][lens[b] - 1] for b in range(2)]))
        for g, (out, lse) in graphs:
            g.replay()
            c.compare(out, lse, *part.reference(True))


@pytest.mark.parametrize("n", [1, 90])
def test_on_another_stream_and_twice_at_once(h, n):
    c = Case(h, [n], [2000], 16, 2, 64, False, seed=8).fill()
    q = c.q.cuda()
    want = h.cache_attn(q, c.cache, c.batch)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append([h.cache_attn(q, c.cache, c.batch) for _ in range(4)])
    torch.cuda.synchronize()
    for o in outs:
        for x in o:
            assert torch.equal(x, want)  # the order of the sums does not depend on timing


@pytest.mark.parametrize("n", [1, 150])
def test_bad_numbers_are_reported_and_not_followed(h, n):
    from pika_h3_flex_b200 import _lib

    c = Case(h, [n], [200], 2, 2, 16, False).fill()
    k = torch.zeros(n, 2, D, dtype=torch.bfloat16, device="cuda")
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    good = (c.batch.pages, c.batch.lengths, c.batch.starts)
    wrong_page = good[0].clone()
    wrong_page[0, 12] = 10 ** 6
    negative = good[0].clone()
    negative[0, 12] = -5
    for parts in ((wrong_page, good[1], good[2]), (negative, good[1], good[2]), (good[0], dev([10 ** 8]), good[2]),
                  (good[0], dev([-3]), good[2]), (good[0], good[1], dev([0, n + 50])), (good[0], good[1], dev([n, 0])),
                  (good[0], good[1], dev([-4, n]))):
        batch = h.CacheBatch(*parts)
        for call in (lambda s: h.cache_write(c.cache, batch, k, k, status_word=s),
                     lambda s: h.cache_read(c.cache, batch, n, status_word=s),
                     lambda s: h.cache_attn(c.q.cuda(), c.cache, batch, status_word=s)):
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            call(status)
            if parts[2] is good[2] or h.read_status(status) != 0:  # offsets that decrease name no row: nothing to move
                with pytest.raises(_lib.H3AError) as e:
                    h.check_status(status)
                assert e.value.status == _lib.H3A_ERR_INDEX
            call(None)


def test_nothing_runs_while_the_status_word_is_set(h):
    c = Case(h, [1], [30], 2, 2, 16, False).fill()
    status = torch.full((1,), 7, dtype=torch.int32, device="cuda")
    out = torch.full((1, 2, D), 4.0, dtype=torch.bfloat16, device="cuda")
    h.cache_attn(c.q.cuda(), c.cache, c.batch, out=out, status_word=status)
    kv = tuple(torch.full((1, 2, D), 4.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    h.cache_read(c.cache, c.batch, out=kv, status_word=status)
    assert (out == 4).all() and (kv[0] == 4).all() and (kv[1] == 4).all()


def test_refusals(h):
    c = Case(h, [2], [20], 4, 2, 16, True).fill()
    q, kv = c.q.cuda(), torch.zeros(2, 2, D, dtype=torch.bfloat16, device="cuda")
    from pika_h3_flex_b200 import _lib

    with pytest.raises(ValueError, match="not a multiple"):
        h.cache_attn(q[:, :3], c.cache, c.batch)
    with pytest.raises(TypeError):
        h.cache_attn(q.half(), c.cache, c.batch)
    with pytest.raises(ValueError, match="q's shape"):
        h.cache_attn(q, c.cache, c.batch, out=torch.empty(3, 4, D, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(_lib.H3AError) as e:
        h.cache_attn(q, c.cache, c.batch, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))
    assert e.value.status == _lib.H3A_ERR_WORKSPACE
    with pytest.raises(ValueError, match="heads"):
        h.cache_write(c.cache, c.batch, kv[:, :1], kv[:, :1])
    with pytest.raises(ValueError, match="disagree"):
        h.cache_write(c.cache, c.batch, kv, kv[:1])
    with pytest.raises(ValueError, match="rows or out"):
        h.cache_read(c.cache, c.batch)
    with pytest.raises(_lib.H3AError) as e:  # rows that are not 16-byte aligned
        odd = torch.zeros(2, 2, D + 4, dtype=torch.bfloat16, device="cuda")
        h.cache_write(c.cache, c.batch, odd[:, :, :D], odd[:, :, :D])
    assert e.value.status == _lib.H3A_ERR_ALIGN
    with pytest.raises(ValueError, match="go together"):
        h.KVCache(c.cache.k, c.cache.v, c.cache.k_exp)
    with pytest.raises(TypeError):
        h.KVCache(c.cache.k.float(), c.cache.v.float())
    with pytest.raises(ValueError, match="multiple of 16"):
        h.KVCache.empty(3, 20, 2)
    with pytest.raises(TypeError, match="int32"):
        h.CacheBatch(c.batch.pages.long(), c.batch.lengths, c.batch.starts)
    with pytest.raises(ValueError):
        h.CacheBatch(c.batch.pages, c.batch.lengths, c.batch.starts[:1])
    with pytest.raises(_lib.H3AError) as e:  # one row for all
        h.cache_attn(q[:1].expand(2, 4, D), c.cache, c.batch)
    assert e.value.status == _lib.H3A_ERR_ALIGN
    with pytest.raises(_lib.H3AError) as e:
        h.cache_attn(q, c.cache, c.batch, max_new=-1)
    assert e.value.status == _lib.H3A_ERR_ARG
    need = h.cache_attn_workspace_bytes(c.cache, c.batch, 2, 4)
    with pytest.raises(_lib.H3AError) as e:
        h.cache_attn(q, c.cache, c.batch, workspace=torch.empty(need + 16, dtype=torch.uint8, device="cuda")[16:])
    assert e.value.status == _lib.H3A_ERR_ALIGN
    with pytest.raises(_lib.H3AError) as e:
        h.cache_attn(q, c.cache, c.batch, out=q)
    assert e.value.status == _lib.H3A_ERR_ARG
    assert h.cache_attn(q[:0], c.cache, c.batch).shape == (0, 4, D)
    assert h.cache_read(c.cache, c.batch, 0)[0].shape == (0, 2, D)
