"""The paged cache: tables against an allocator written out in Python, rows against indexing, the attention of one token
against the formula in 64 bits, and the three together as a server uses them."""
import math

import pytest
import torch
import torch.nn.functional as F

import forgetting_transformer_b200 as fox

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ tables
class Allocator:
    """What page_tables and release_pages do, request by request."""

    def __init__(self, R, width, pages, page):
        self.page, self.width = page, width
        self.table = [[-1] * width for _ in range(R)]
        self.lengths, self.free = [0] * R, list(range(pages))

    def pages(self, n):
        return -(-n // self.page)

    def extend(self, new, max_tokens):
        starts, granted, tokens, short = [0], [], [], False
        for r, n in enumerate(new):
            n = max(n, 0)
            old = self.lengths[r]
            fits = self.pages(old + n) <= self.width and starts[-1] + n <= max_tokens
            need = self.pages(old + n) - self.pages(old) if fits else 0
            if need and (short or need > len(self.free)):
                short, ok = True, False         # (those behind get no page either, so that the order is kept)
            else:
                ok = fits
            if ok:
                for j in range(self.pages(old), self.pages(old + n)):
                    self.table[r][j] = self.free.pop()
                self.lengths[r] = old + n
            granted.append(n if ok else 0)
            for t in range(old, old + n):
                tokens.append((r, t, self.table[r][t // self.page] * self.page + t % self.page if ok else -1))
            starts.append(starts[-1] + n)
        tokens = (tokens + [(-1, 0, -1)] * max_tokens)[:max_tokens]
        return starts, granted, tokens

    def crop(self, keep):
        for r, n in enumerate(keep):
            n = min(max(n, 0), self.lengths[r])
            for j in range(self.pages(n), self.pages(self.lengths[r])):
                self.free.append(self.table[r][j])
                self.table[r][j] = -1
            self.lengths[r] = n


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("R,width,pages,page,most,max_tokens", [
    (1, 2, 5, 16, 40, 20), (3, 5, 7, 16, 40, 60), (40, 8, 60, 16, 120, 1500), (1025, 5, 1100, 32, 9, 1700), (2500, 3, 2400, 16, 9, 8192),
    (7, 400, 700, 16, 4000, 9000), (300, 20, 800, 64, 600, 23000)])
def test_tables_over_many_calls(R, width, pages, page, most, max_tokens):
    """Extensions and cuts in turn, with requests that outgrow their row, the packed batch or the pool."""
    rng = __import__("random").Random(R + pages)
    a = Allocator(R, width, pages, page)
    lengths, table = i32([0] * R), torch.full((R, width + 3), -1, dtype=torch.int32, device="cuda")[:, :width]
    free, num_free = i32(a.free), i32([pages])
    refused = 0
    for step in range(8):
        new = [rng.choice([0, 1, 1, rng.randint(0, most)]) for _ in range(R)]
        if step == 3:
            new[0] = -5
        inplace = step % 2 == 1
        t = fox.page_tables(lengths, i32(new), table, free, num_free, page, max_tokens, inplace=inplace)
        starts, granted, tokens = a.extend(new, max_tokens)
        if inplace:
            assert t.lengths is lengths and t.num_free is num_free
        lengths, num_free = t.lengths.clone(), t.num_free.clone()
        refused += sum(max(n, 0) for n in new) > sum(granted)
        assert t.starts.tolist() == starts and t.granted.tolist() == granted
        assert lengths.tolist() == a.lengths and num_free.tolist() == [len(a.free)]
        assert list(zip(t.requests.tolist(), t.positions.tolist(), t.slots.tolist())) == tokens
        assert table.tolist() == a.table
        if step % 3 == 2:
            keep = [rng.choice([0, n, n // 2, n + 7, -1]) for n in a.lengths]
            fox.release_pages(lengths, i32(keep), table, free, num_free, page)
            a.crop(keep)
            assert lengths.tolist() == a.lengths and table.tolist() == a.table
            assert num_free.tolist() == [len(a.free)] and free[:len(a.free)].tolist() == a.free
    owned = [p for row in a.table for p in row if p >= 0]
    assert sorted(owned + a.free) == list(range(pages))
    assert refused or R == 1


def test_tables_without_tokens():
    lengths, table, free, num_free = i32([5, 0]), i32([[3, -1], [-1, -1]]), i32([0, 1, 2]), i32([3])
    t = fox.page_tables(lengths, i32([0, 0]), table, free, num_free, 16, 0)
    assert t.lengths.tolist() == [5, 0] and t.num_free.tolist() == [3] and t.starts.tolist() == [0, 0, 0] and t.slots.numel() == 0
    # counts outside their range are taken as its ends: nothing is read or written beyond the arrays
    t = fox.page_tables(i32([-3, 0]), i32([4, 20]), table, free, i32([77]), 16, 40)
    assert t.lengths.tolist() == [4, 20] and t.num_free.tolist() == [0] and table.tolist() == [[2, -1], [1, 0]]


# ------------------------------------------------------------------ rows
@pytest.mark.parametrize("T,H,Hk,D,page", [(1, 1, 1, 16, 16), (5, 6, 2, 32, 16), (61, 16, 16, 128, 32), (700, 4, 4, 64, 64), (20000, 3, 1, 64, 128)])
@pytest.mark.parametrize("gates", ["log", "bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_into_pages(T, H, Hk, D, page, gates, dtype):
    """Rows go where their slots say, the rest of the pool stays; tokens without a slot and strided inputs.  A logit's log
    sigmoid is a sum of fp32 functions good to a few ulp: 2^-21 of its value."""
    P = T // page + 9
    pool = [torch.randn(P, Hk, page, D, generator=gen(1)).to(dtype).cuda(), torch.randn(P, Hk, page, D, generator=gen(2)).to(dtype).cuda(),
            torch.randn(P, H, page, generator=gen(3)).cuda()]
    row = torch.randn(T, 2 * Hk * D + 8, generator=gen(4)).to(dtype).cuda()
    k, v = row[:, :Hk * D].view(T, Hk, D), row[:, Hk * D + 8:].view(T, Hk, D)
    g = torch.randn(H, T, generator=gen(5)).cuda().mul(5).t()
    if gates != "log":
        g = g.to({"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[gates])
    slots = torch.randperm(P * page, generator=gen(6))[:T]
    slots[::7] = -1
    slots[3::11] = P * page
    slots[5::13] = 2 ** 31 - 1
    want = [t.clone() for t in pool]
    on = ((slots >= 0) & (slots < P * page)).nonzero()[:, 0].cuda()
    at = slots.cuda()[on]
    want[0][at // page, :, at % page] = k[on]
    want[1][at // page, :, at % page] = v[on]
    lf = g if gates == "log" else F.logsigmoid(g.double())
    want[2] = want[2].double()
    want[2][at // page, :, at % page] = lf[on].double()
    fox.paged_update(*pool, k, v, g, slots.cuda() if T % 2 else slots.int().cuda(), gate_is_logit=gates != "log")
    assert torch.equal(pool[0], want[0]) and torch.equal(pool[1], want[1])
    assert ((pool[2].double() - want[2]).abs() <= (0 if gates == "log" else 2 ** -21) * want[2].abs()).all()


def test_rows_into_views_of_a_pool():
    """Keys and values interleaved in one tensor, gates with a stride, slots with a stride; no tokens at all."""
    both = torch.zeros(6, 2, 3, 16, 64, dtype=torch.bfloat16, device="cuda")
    gates = torch.zeros(6, 4, 3, 16, device="cuda")[:, 1]
    k, v = [torch.randn(10, 3, 64, generator=gen(i)).bfloat16().cuda() for i in range(2)]
    g = -torch.rand(10, 3, generator=gen(2)).cuda()
    slots = torch.randperm(96, generator=gen(3))[:20].int().cuda()[::2]
    fox.paged_update(both[:, 0], both[:, 1], gates, k, v, g, slots)
    p, r = slots.long() // 16, slots.long() % 16
    assert torch.equal(both[p, 0, :, r], k) and torch.equal(both[p, 1, :, r], v) and torch.equal(gates[p, :, r], g)
    assert both.float().abs().sum() == k.float().abs().sum() + v.float().abs().sum()
    before = both.clone()
    fox.paged_update(both[:, 0], both[:, 1], gates, k[:0], v[:0], g[:0], slots[:0])
    assert torch.equal(before, both)


# ------------------------------------------------------------------ attention
def reference(q, kp, vp, gp, table, lengths, scale):
    """out and log-sum-exp in 64 bits, and a bound of what fp32 work and 16-bit weights may differ by, before the last rounding.

    A logit's products are summed in fp32 (2^-19 of the sum of their sizes), its bias is a running sum of n / 16 + 40 additions
    (that many times 2^-24 of its size); a weight is off by the logit's error, by 2^-20 of its own, and by 2^-16 (bf16; fp16
    less) of what its two 16-bit parts leave; the sums over keys follow: E."""
    R, H, D = q.shape
    Hk, page = kp.shape[1], kp.shape[2]
    out, lse, tol = [torch.zeros(*s, dtype=torch.float64, device=q.device) for s in ((R, H, D), (R, H), (R, H, D))]
    for r in range(R):
        n = int(lengths[r])
        if n == 0:
            lse[r] = -math.inf
            continue
        ids = table[r, :-(-n // page)].long()
        there = ((ids >= 0) & (ids < kp.shape[0])).repeat_interleave(page)[:n]
        ids = ids.clamp(0, kp.shape[0] - 1)
        k, v = [t[ids].transpose(0, 1).flatten(1, 2)[:, :n].double().repeat_interleave(H // Hk, 0) for t in (kp, vp)]
        g = torch.where(there, gp[ids].transpose(0, 1).flatten(1, 2)[:, :n].double(), 0.0)
        if not there.all():
            k, v = [torch.where(there[:, None], t, 0.0) for t in (k, v)]
        behind = torch.cat([g[:, 1:], g.new_zeros(H, 1)], 1).flip(1).cumsum(1).flip(1)
        qr = q[r].double()[:, None]
        u = torch.where(there, (k * qr).sum(-1) * scale + behind, -math.inf)
        e = (k.abs() * qr.abs()).sum(-1) * abs(scale) * 2 ** -19 + torch.where(u > -math.inf, behind, 0.0).abs() * (n / 16 + 40) * 2 ** -24 + 2 ** -16
        p = u.softmax(-1) if there.any() else torch.zeros_like(u)
        out[r] = (p[..., None] * v).sum(1)
        lse[r] = u.logsumexp(-1)
        pe = p * torch.where(p > 0, e, 0.0)
        tol[r] = (pe[..., None] * v.abs()).sum(1) + pe.sum(-1, keepdim=True) * out[r].abs()
    return out, lse, tol


def pool_of(seed, lengths, H, Hk, D, page, dtype, mu=3.0, width=None, extra=3):
    """A pool whose unused rows and pages are NaN, and a table in a random order."""
    have = [-(-n // page) for n in lengths]
    width = width or max(1, max(have))
    P = sum(have) + extra
    nan = lambda *s, **kw: torch.full(s, math.nan, device="cuda", **kw)
    kp, vp, gp = nan(P, Hk, page, D, dtype=dtype), nan(P, Hk, page, D, dtype=dtype), nan(P, H, page)
    order = torch.randperm(P, generator=gen(seed)).int()
    table = torch.full((len(lengths), width), 2 ** 30, dtype=torch.int32)      # (nothing looks at what is behind a length)
    at = 0
    for r, n in enumerate(lengths):
        table[r, :have[r]] = order[at:at + have[r]]
        at += have[r]
    table = table.cuda()
    for r, n in enumerate(lengths):
        if n:
            t = torch.arange(n, device="cuda")
            p, row = table[r].long()[t // page], t % page
            g = gen(seed + 17 * r + 1)
            kp[p, :, row] = torch.randn(n, Hk, D, generator=g).to(dtype).cuda()
            vp[p, :, row] = torch.randn(n, Hk, D, generator=g).to(dtype).cuda()
            gp[p, :, row] = F.logsigmoid(torch.randn(n, H, generator=g) + mu).cuda()
    return kp, vp, gp, table, i32(lengths)


def check(q, kp, vp, gp, table, lengths, scale=None, got=None):
    scale_ = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    out, L = fox.paged_forgetting_attention(q, kp, vp, gp, table, lengths, sm_scale=scale, return_log_normalizer=True) if got is None else got
    ref, lse, tol = reference(q, kp, vp, gp, table, lengths, scale_)
    half = torch.finfo(q.dtype).eps / 2
    err = (out.double() - ref).abs()
    bound = half * ref.abs() + tol + (2 ** -25 if q.dtype == torch.float16 else 0)
    assert out.dtype == q.dtype and (err <= bound).all(), ((err - bound).max().item(), err.max().item())
    live = lse > -math.inf
    assert torch.equal(live, L > -math.inf)
    n = lengths.max().item()
    assert ((L.double() - lse)[live].abs() <= 2 ** -14 + 2 ** -18 * lse[live].abs() + (n / 16) * 2 ** -24).all()
    return out


def queries(seed, R, H, D, dtype):
    return torch.randn(R, H, D, generator=gen(seed)).to(dtype).cuda()


@pytest.mark.parametrize("H,Hk,D,page", [(2, 2, 64, 16), (3, 3, 128, 32), (5, 5, 16, 16), (4, 4, 32, 64), (8, 2, 64, 128), (14, 2, 128, 16),
                                         (8, 1, 16, 16), (20, 2, 32, 16), (9, 1, 64, 32), (33, 3, 128, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lengths_around_tiles_and_pages(H, Hk, D, page, dtype):
    """One key to a few tiles, ends inside and at the ends of tiles and pages, places without a request among them."""
    lengths = [1, 0, 15, 16, 17, 31, 32, 33, 0, 47, 64, 65, 127, 128, 129, 200, 255, 257, 300, 0]
    pool = pool_of(H + D, lengths, H, Hk, D, page, dtype)
    out = check(queries(1, len(lengths), H, D, dtype), *pool)
    assert out[[1, 8, 19]].abs().max() == 0


@pytest.mark.parametrize("lengths,H,Hk,D,page,dtype,mu", [
    ([70001], 1, 1, 64, 16, torch.bfloat16, 6.0),          # one unit in hundreds of ranges
    ([5000, 3, 9001], 2, 2, 128, 64, torch.float16, 4.0),
    ([20000], 8, 1, 64, 256, torch.bfloat16, 5.0),
    ([1300] * 3 + [40] * 200, 6, 3, 64, 16, torch.float16, 1.0),   # ranges of many units
    ([5] * 700, 4, 4, 32, 16, torch.bfloat16, 2.0),
    ([2048, 1], 24, 24, 16, 1024, torch.float16, 3.0),
    ([33000], 16, 2, 128, 32, torch.bfloat16, 6.0),
    ([9] * 1300 + [0] * 1300, 1, 1, 64, 16, torch.bfloat16, 2.0),  # more requests than threads
    ([65536], 3, 3, 64, 65536, torch.bfloat16, 7.0),
])
def test_long_and_many(lengths, H, Hk, D, page, dtype, mu):
    pool = pool_of(len(lengths), lengths, H, Hk, D, page, dtype, mu=mu)
    check(queries(2, len(lengths), H, D, dtype), *pool)


def test_scale_strides_and_one_gate_for_all_heads():
    """Views: q out of a projection's row, pages of one tensor, a table that is a part of a wider one, gates alike for all heads."""
    lengths = [40, 100, 7]
    kp, vp, gp, table, n = pool_of(5, lengths, 4, 2, 64, 16, torch.bfloat16)
    both = torch.empty(kp.shape[0], 2, 3, 16, 72, dtype=torch.bfloat16, device="cuda")[:, :, :2, :, :64]
    both[:, 0], both[:, 1] = kp, vp
    wide = torch.full((3, 50), 7, dtype=torch.int32, device="cuda")
    wide[:, 9:9 + table.shape[1]] = table
    row = queries(3, 3, 9, 64, torch.bfloat16)
    view = row[:, 2:6]
    gates = gp[:, :1].expand(-1, 4, -1)
    got = fox.paged_forgetting_attention(view, both[:, 0], both[:, 1], gates, wide[:, 9:9 + table.shape[1]], n, sm_scale=0.3,
                                         return_log_normalizer=True)
    check(view, kp, vp, gates, table, n, 0.3, got)
    odd = torch.zeros(3 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 4, 64)      # (copied: no 16-byte rows)
    odd.copy_(view)
    assert torch.equal(fox.paged_forgetting_attention(odd, kp, vp, gates, table, n, sm_scale=0.3), got[0])


@pytest.mark.parametrize("value", [-math.inf, -3.4028234663852886e38, -1e4, 0.0])
def test_gates_that_close_or_never_do(value):
    """Gates of minus infinity, of the type's lowest value, closed but for the last key, and open: no NaN from sums of them, the
    keys before a closed gate without a share."""
    lengths = [300, 1, 33, 5000]
    kp, vp, gp, table, n = pool_of(9, lengths, 2, 2, 64, 16, torch.bfloat16)
    for r, ln in enumerate(lengths):
        t = torch.arange(ln, device="cuda")
        shut = t % 37 == 36 if value else t >= 0
        p, row = table[r].long()[t // 16], t % 16
        gp[p[shut], 0, row[shut]] = value
    check(queries(4, 4, 2, 64, torch.bfloat16), kp, vp, gp, table, n)


def test_infinite_and_nan_values():
    """A NaN key or value reaches its own request and heads only, also where the request is cut into ranges; values of minus
    infinity behind a length never."""
    lengths = [3000, 3000]
    kp, vp, gp, table, n = pool_of(11, lengths, 4, 2, 64, 16, torch.float16)
    q = queries(5, 2, 4, 64, torch.float16)
    clean = fox.paged_forgetting_attention(q, kp, vp, gp, table, n)
    assert clean.isfinite().all()
    kp[table[0, 3].long(), 1, 5] = math.nan
    vp[table[1, 100].long(), 0, 7, 9] = math.nan
    out = fox.paged_forgetting_attention(q, kp, vp, gp, table, n)
    assert out[0, 2:].isnan().all() and torch.equal(out[0, :2], clean[0, :2])
    assert out[1, :2, 9].isnan().all() and torch.equal(out[1, 2:], clean[1, 2:]) and out[1, :2, :9].isfinite().all()
    gp[table[0, 3].long(), 0, 5] = math.nan
    assert fox.paged_forgetting_attention(q, kp, vp, gp, table, n)[0, 0].isnan().all()


def test_entries_outside_the_pool_and_lengths_outside_the_table():
    """A page that is not there leaves its keys out; a length beyond the table's entries ends with them, one below zero is zero.
    (The kernel compares every entry with the pool's size before it forms an address from it.)"""
    lengths = [100, 50, 64, 48]
    kp, vp, gp, table, n = pool_of(13, lengths, 2, 1, 64, 16, torch.bfloat16, width=7)
    table[0, 2], table[1, 3], table[2, :4] = -1, kp.shape[0], 2 ** 31 - 1
    q = queries(6, 4, 2, 64, torch.bfloat16)
    out = check(q, kp, vp, gp, table, n)
    assert out[2].abs().max() == 0
    narrow = table[:, :3].contiguous()
    a = fox.paged_forgetting_attention(q[3:], kp, vp, gp, narrow[3:], i32([2 ** 31 - 1]))
    assert torch.equal(a, fox.paged_forgetting_attention(q[3:], kp, vp, gp, table[3:], n[3:]))
    assert fox.paged_forgetting_attention(q[:1], kp, vp, gp, table[:1], i32([-4])).abs().max() == 0
    none = fox.paged_forgetting_attention(q[:0], kp, vp, gp, table[:0], n[:0])
    assert none.shape == (0, 2, 64)
    out, L = fox.paged_forgetting_attention(q, kp, vp, gp, table[:, :0], n, return_log_normalizer=True)
    assert out.abs().max() == 0 and (L == -math.inf).all()


def test_pages_beyond_four_gigabytes():
    """Pages whose elements pass 32 bits: the last page of a pool of 2^31 elements and more of each."""
    P, page, D = 2 ** 31 // (128 * 128) + 2, 128, 128
    kp, vp = [torch.zeros(P, 1, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    gp = torch.zeros(P, 1, page, device="cuda")
    k, v = [torch.randn(200, 1, D, generator=gen(i)).bfloat16().cuda() for i in range(2)]
    table = i32([[P - 1, P - 2]])
    t = torch.arange(200, device="cuda")
    slots = table[0].long()[t // page] * page + t % page
    fox.paged_update(kp, vp, gp, k, v, -torch.rand(200, 1, generator=gen(3)).cuda(), slots)
    assert torch.equal(kp[P - 1, 0], k[:128, 0]) and torch.equal(vp[P - 2, 0, :72], v[128:, 0])
    check(queries(7, 1, 1, D, torch.bfloat16), kp, vp, gp, table, i32([200]))


def test_same_page_in_two_requests():
    """Requests may share pages (a common beginning), and name a page twice."""
    kp, vp, gp, table, n = pool_of(15, [64, 64], 2, 2, 64, 16, torch.bfloat16)
    table[1, :2] = table[0, :2]
    table[1, 3] = table[1, 2]
    check(queries(8, 2, 2, 64, torch.bfloat16), kp, vp, gp, table, n)


def test_very_wide_tables():
    """Tables whose rows could hold more tiles than are counted at a time: the requests go in several launches."""
    lengths = [40, 0, 1000, 17, 3, 0, 5000, 64, 65, 1]
    kp, vp, gp, table, n = pool_of(40, lengths, 16, 16, 64, 64, torch.bfloat16)
    wide = torch.full((len(lengths), 2 ** 21), -7, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    q = queries(9, len(lengths), 16, 64, torch.bfloat16)
    got = fox.paged_forgetting_attention(q, kp, vp, gp, wide, n, return_log_normalizer=True)
    check(q, kp, vp, gp, table, n, None, got)


def test_inference_mode():
    cache = fox.PagedFgateCache(1, 8, 16, 2, 64, 2, 50)
    with torch.inference_mode():
        t = cache.extend(i32([3, 20]), 30)
        k = torch.randn(30, 2, 64, generator=gen(1)).bfloat16().cuda()
        cache.update(0, k, k, -torch.ones(30, 2, device="cuda"), t.slots)
        out = cache.attend(0, k[:2])
        cache.release(torch.tensor([True, False], device="cuda"))
    check(k[1:2], *cache[0], cache.block_table[1:], cache.lengths[1:], None,
          (out[1:], fox.paged_forgetting_attention(k[1:2], *cache[0], cache.block_table[1:], cache.lengths[1:], return_log_normalizer=True)[1]))
    assert cache.lengths.tolist() == [0, 20] and cache.num_free.tolist() == [6]


def test_streams_and_graphs():
    """Two captured calls on streams of their own, replayed side by side on new values, against plain calls; results of a call
    do not change from one to the next."""
    cases = []
    for i, lengths in enumerate(([4000, 17, 900], [333, 5001, 2])):
        pool = pool_of(20 + i, lengths, 4, 4, 64, 16, torch.bfloat16)
        cases.append((queries(i, 3, 4, 64, torch.bfloat16), *pool))
    graphs = []
    for c in cases:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            fox.paged_forgetting_attention(*c)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                out = fox.paged_forgetting_attention(*c)
        graphs.append((s, g, out))
    torch.cuda.synchronize()
    for i, c in enumerate(cases):
        c[0].copy_(queries(30 + i, 3, 4, 64, torch.bfloat16))
        c[5].copy_(i32([[3999, 10, 0], [300, 4000, 1]][i]))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, g, _ in graphs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c, (_, _, out) in zip(cases, graphs):
        want = fox.paged_forgetting_attention(*c)
        assert torch.equal(out, want)
        check(*c)


# ------------------------------------------------------------------ together
def test_serving_run():
    """Prompts of different lengths come in together, tokens are generated for all, one request ends and another takes its
    place: at every step each request's attention is that of its own history, kept here as plain tensors."""
    H, Hk, D, page, R, layers = 4, 2, 64, 16, 5, 2
    dtype = torch.bfloat16
    cache = fox.PagedFgateCache(layers, 60, page, H, D, R, 300, num_kv_heads=Hk, dtype=dtype)
    rot, (wq, wk) = fox.RotaryEmbedding(D), [1 + 0.1 * torch.randn(D, generator=gen(i)).cuda() for i in range(2)]
    hist = [[[] for _ in range(R)] for _ in range(layers)]
    alive = [0] * R

    def step(new, seed):
        total = sum(new) + 3                        # (a packed batch with room behind its last token)
        t = cache.extend(i32(new), total)
        assert t.granted.tolist() == new
        starts = t.starts.tolist()
        for layer in range(layers):
            g = gen(seed * 10 + layer)
            q = torch.randn(total, H, D, generator=g).to(dtype).cuda()
            k = torch.randn(total, Hk, D, generator=g).to(dtype).cuda()
            v = torch.randn(total, Hk, D, generator=g).to(dtype).cuda()
            logit = (torch.randn(total, H, generator=g) + 3).to(dtype).cuda()
            q, k = rot.norm(q, k, wq, wk, t.positions)
            cache.update(layer, k, v, logit, t.slots, gate_is_logit=True)
            lf = F.logsigmoid(logit.double())
            for r in range(R):
                a, b = starts[r], starts[r + 1]
                if b > a:
                    hist[layer][r].append((k[a:b], v[a:b], lf[a:b]))
            last = torch.tensor([max(x - 1, 0) for x in starts[1:]], device="cuda")
            out = cache.attend(layer, q[last])
            for r in range(R):
                if not alive[r] + new[r]:
                    assert out[r].abs().max() == 0
                    continue
                kk, vv, gg = [torch.cat(x).double() for x in zip(*hist[layer][r])]
                n = len(kk)
                assert n == int(cache.lengths[r])
                kk, vv = [x.repeat_interleave(H // Hk, 1) for x in (kk, vv)]
                behind = gg.flip(0).cumsum(0).flip(0) - gg
                u = torch.einsum("hd,nhd->hn", q[last[r]].double(), kk) / 8 + behind.t()
                p = u.softmax(-1)
                ref = torch.einsum("hn,nhd->hd", p, vv)
                size = torch.einsum("hn,nhd->hd", p, vv.abs())
                # (gates are kept in fp32: a bias of up to 300 of them is off by 300 * 2^-21 of its size, at most 2^-9 where a
                #  key's share is above e^-12; 2^-12 covers the mean over keys, whose biases near the end are exact)
                assert ((out[r].double() - ref).abs() <= 2 ** -8 * ref.abs() + 2 ** -12 * size).all()
        for r in range(R):
            alive[r] += new[r]
    step([33, 1, 0, 120, 16], 1)
    for i in range(4):
        step([1, 1, 0, 1, 1], 2 + i)
    end = torch.tensor([False, False, False, True, False], device="cuda")
    free = int(cache.num_free)
    cache.release(end)
    assert int(cache.num_free) == free + 8 and int(cache.lengths[3]) == 0
    alive[3] = 0
    for layer in hist:
        layer[3] = []
    step([1, 0, 70, 50, 1], 9)
    step([1, 1, 1, 1, 1], 10)
    # a request's history goes to the full operator as it is
    k, v, g = cache.history(0, 2, int(cache.lengths[2]))
    kk, vv, gg = [torch.cat(x) for x in zip(*hist[0][2])]
    assert torch.equal(k[0].transpose(0, 1), kk) and torch.equal(v[0].transpose(0, 1), vv)
    q = torch.randn(1, H, 1, D, generator=gen(99)).to(dtype).cuda()
    with torch.no_grad():
        full = fox.forgetting_attention(q, k.repeat_interleave(2, 1), v.repeat_interleave(2, 1), g, head_first=True)
    here = cache.attend(0, q[:, :, 0].expand(R, -1, -1))[2]
    assert (full[0, :, 0].double() - here.double()).abs().max() <= 2 ** -7 * full.double().abs().max()


def test_generation_step_in_a_graph():
    """A whole step, tables included, captured once and replayed: every replay adds a token to each request."""
    H, D, R = 4, 64, 3
    cache = fox.PagedFgateCache(1, 40, 16, H, D, R, 200)
    x = torch.zeros(R, 3 * H * D, dtype=torch.bfloat16, device="cuda")
    logit = torch.full((R, H), 3.0, device="cuda")
    one = i32([1] * R)

    def step():
        t = cache.extend(one, R)
        q, k, v = x.view(R, 3, H, D).unbind(1)
        cache.update(0, k, v, logit, t.slots, gate_is_logit=True)
        return cache.attend(0, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        cache.release(torch.ones(R, dtype=torch.bool, device="cuda"))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step()
    torch.cuda.current_stream().wait_stream(side)
    cache.lengths.zero_()
    rows = []
    for i in range(40):
        x.copy_(torch.randn(R, 3 * H * D, generator=gen(i)))
        g.replay()
        rows.append(x.clone())
        assert cache.lengths.tolist() == [i + 1] * R
    assert torch.equal(out, check(x.view(R, 3, H, D)[:, 0], *cache[0], cache.block_table, cache.lengths))
    k = torch.stack(rows).view(40, R, 3, H, D)[:, :, 1]
    for r in range(R):
        assert torch.equal(cache.history(0, r, 40)[0][0].transpose(0, 1), k[:, r])


# ------------------------------------------------------------------ ends of ranges
@pytest.mark.parametrize("pages,some_are_refused", [(9000, False), (3000, True)])
def test_tables_of_more_requests_than_a_block_keeps(pages, some_are_refused):
    """More requests than the placing kernel holds in shared memory, and more tokens than the scanning CTA places by itself."""
    R, width, page, most, max_tokens = 5003, 4, 16, 12, 23000
    rng = __import__("random").Random(R + pages)
    a = Allocator(R, width, pages, page)
    lengths, table = i32([0] * R), torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    free, num_free = i32(a.free), i32([pages])
    refused = False
    for step in range(6):
        new = [rng.choice([0, 1, 1, rng.randint(0, most)]) for _ in range(R)]
        t = fox.page_tables(lengths, i32(new), table, free, num_free, page, max_tokens, inplace=step % 2 == 1)
        starts, granted, tokens = a.extend(new, max_tokens)
        lengths, num_free = t.lengths, t.num_free
        refused = refused or granted != new
        assert t.starts.tolist() == starts and t.granted.tolist() == granted
        assert lengths.tolist() == a.lengths and num_free.tolist() == [len(a.free)]
        assert list(zip(t.requests.tolist(), t.positions.tolist(), t.slots.tolist())) == tokens
        assert table.tolist() == a.table
        if step == 3:
            keep = [rng.choice([0, n, n // 2, n + 7, -1]) for n in a.lengths]
            fox.release_pages(lengths, i32(keep), table, free, num_free, page)
            a.crop(keep)
            assert lengths.tolist() == a.lengths and table.tolist() == a.table and free[:len(a.free)].tolist() == a.free
    assert refused == some_are_refused


@pytest.mark.parametrize("T,H,Hk,D,page", [(18944, 2, 2, 16, 16), (19003, 6, 3, 32, 64), (19111, 5, 5, 128, 32), (25001, 24, 24, 64, 64)])
@pytest.mark.parametrize("gates", ["log", "fp32"])
def test_rows_of_long_prompts_into_pages(T, H, Hk, D, page, gates):
    """Calls large enough for eight tokens ahead (16 tiles of 8 tokens to an SM), the last tile ragged."""
    assert -(-T // 8) >= 16 * 148
    test_rows_into_pages(T, H, Hk, D, page, gates, torch.bfloat16)


def test_packed_batch_by_its_tables():
    """The queries of a packed batch found on the device, by the tables' own starts: a prompt, single tokens, a place without a request, a
    request with nothing new, and one that is refused and keeps what it has."""
    H, Hk, D, R = 4, 2, 64, 6
    cache = fox.PagedFgateCache(1, 20, 16, H, D, R, 200, num_kv_heads=Hk)

    def step(new, room, seed):
        t = cache.extend(i32(new), room)
        k, v = [torch.randn(room, Hk, D, generator=gen(seed + i)).bfloat16().cuda() for i in range(2)]
        cache.update(0, k, v, -torch.rand(room, H, generator=gen(seed + 2)).cuda(), t.slots)
        return t
    step([40, 0, 7, 33, 1, 5], 90, 1)
    new = [1, 0, 60, 1, 0, 400]             # (the last is longer than its row)
    t = step(new, 70, 5)
    q = torch.randn(70, H, D, generator=gen(9)).bfloat16().cuda()
    last = (t.starts[1:].long() - 1).clamp(0, q.shape[0] - 1)
    out = cache.attend(0, q[last])
    assert t.granted.tolist() == [1, 0, 60, 1, 0, 0] and cache.lengths.tolist() == [41, 0, 67, 34, 1, 5]
    assert last.tolist()[:4] == [0, 0, 60, 61]
    L = fox.paged_forgetting_attention(q[last], *cache[0], cache.block_table, cache.lengths, return_log_normalizer=True)[1]
    check(q[last], *cache[0], cache.block_table, cache.lengths, None, (out, L))
    assert not out[1].any()
