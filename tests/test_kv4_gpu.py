"""KV4Cache (4-bit paged K/V cache) against a plain implementation in 64 bits."""
import math

import pytest
import torch

from vllm_moet_b200.formats import kv4

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def KV4Cache():
    from vllm_moet_b200.ops.kv4 import KV4Cache
    return KV4Cache


class Batch:
    """Sequences with all their raw keys / values, a page table and the query rows."""

    def __init__(self, lens, news, H, G, D, dtype=torch.bfloat16, seed=0, spare=2, q_scale=1.0, width=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.news, self.H, self.G, self.D, self.dtype = lens, news, H, G, D, dtype
        pages = [-(-n // 64) for n in lens]
        self.n_pages = sum(pages) + spare
        perm = torch.randperm(self.n_pages, generator=g).int()
        self.table = torch.full((len(lens), width or max(max(pages), 1)), -7, dtype=torch.int32)
        at, slots = 0, []
        for b, w in enumerate(pages):
            self.table[b, :w] = perm[at:at + w]
            j = torch.arange(lens[b])
            slots.append(self.table[b, j // 64].long() * 64 + j % 64)
            at += w
        self.slots = torch.cat(slots) if slots else torch.zeros(0, dtype=torch.int64)
        total = sum(lens)
        self.k = (torch.randn(total, H, D, generator=g) * 1.3 + 0.4).to(dtype)
        self.v = torch.randn(total, H, D, generator=g).to(dtype)
        self.q = (torch.randn(sum(news), H * G, D, generator=g) * q_scale).to(dtype)
        self.cu = torch.tensor([0] + news).cumsum(0).int()
        self.seq_lens = torch.tensor(lens, dtype=torch.int32)

    def cache(self, KV4Cache, **kw):
        c = KV4Cache(self.n_pages, self.H, self.D, device=DEV, **kw)
        c.append(self.k.to(DEV), self.v.to(DEV), self.slots.to(DEV))
        return c

    def args(self):
        return self.q.to(DEV), self.cu.to(DEV), self.seq_lens.to(DEV), self.table.to(DEV)

    def held(self, x, exp=-6):
        return kv4.values(*kv4.quantise(x, exp), exp).double()

    def oracle(self, scale, window=0, pages=None):
        """(out, lse, sum p |v| / sum p, positions seen) per row, in 64 bits."""
        T, Hq, D, G = self.q.shape[0], self.H * self.G, self.D, self.G
        out = torch.zeros(T, Hq, D, dtype=torch.float64)
        mag = torch.zeros_like(out)
        lse = torch.full((T, Hq), -math.inf, dtype=torch.float64)
        k, v = self.held(self.k), self.held(self.v)
        at = 0
        for b, (n, m) in enumerate(zip(self.lens, self.news)):
            for i in range(m):
                row, p = int(self.cu[b]) + i, n - m + i
                for h in range(self.H):
                    keys = [j for j in range(max(0, p - window + 1) if window else 0, p + 1)]
                    if pages is not None:
                        ok = set(x for x in pages[row, h].tolist() if x >= 0)
                        keys = [j for j in keys if j // 64 in ok]
                    if not keys:
                        continue
                    idx = torch.tensor(keys) + at
                    s = self.q[row, h * G:(h + 1) * G].double() @ k[idx, h].T * scale
                    pr = torch.softmax(s, -1)
                    out[row, h * G:(h + 1) * G] = pr @ v[idx, h]
                    mag[row, h * G:(h + 1) * G] = pr @ v[idx, h].abs()
                    lse[row, h * G:(h + 1) * G] = torch.logsumexp(s, -1)
            at += n
        return out, lse, mag


def check(got, lse, want, keys):
    """Half an ulp of the output (2^-8 of a bf16 value, 2^-11 of an f16 one), P rounded to f16 (2^-11 of every
    term, and 2^-25 of each of at most `keys` terms that are subnormal), and 2^-11 for the f32 scores, whose
    errors (2^-24 of sums of up to 256 terms of size 2^5 or so) enter the exponent."""
    o, l, mag = want
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -11
    got, lse = got.double().cpu(), lse.double().cpu()
    top = mag.amax(-1, keepdim=True)
    bound = half * o.abs() + (2.0 ** -10 + half * 2.0 ** -10) * mag + keys * 2.0 ** -25 * top + 1e-12
    assert torch.isfinite(got).all()
    assert ((got - o).abs() <= bound).all(), float(((got - o).abs() - bound).max())
    empty = l == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (got[empty] == 0).all()
    assert ((lse - l).abs()[~empty] <= 2.0 ** -11).all()


# ------------------------------------------------------------------------------ write and read
@pytest.mark.parametrize("D,H,dtype", [(64, 3, torch.float16), (128, 2, torch.bfloat16), (256, 1, torch.float16),
                                       (64, 1, torch.bfloat16), (128, 8, torch.float16), (256, 2, torch.bfloat16)])
def test_append_gives_the_golden_bytes_and_bounds(KV4Cache, D, H, dtype):
    g = torch.Generator().manual_seed(D + H)
    T, P = 150, 4
    k = (torch.randn(T, H, D, generator=g) * torch.rand(T, H, D // 16, 1, generator=g).repeat(1, 1, 1, 16).view(T, H, D) * 9).to(dtype)
    v = (torch.randn(T, H, D, generator=g) * 0.02).to(dtype)
    k[5] = 0
    k[7, 0, :16] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6]).to(dtype)
    v[9, 0, 0] = 60000.0                                       # saturates its block
    slots = torch.randperm(P * 64, generator=g)[:T]            # any order; pages partly written
    slots[3] = -1
    c = KV4Cache(P, H, D, device=DEV)
    c.append(k.to(DEV), v.to(DEV), slots.to(DEV))
    kc = torch.zeros(P * 64, H, D, dtype=torch.uint8)
    ks = torch.zeros(P * 64, H, D // 16, dtype=torch.uint8)
    vc, vs = kc.clone(), ks.clone()
    live = slots >= 0
    a, b = kv4.quantise(k)
    kc[slots[live]], ks[slots[live]] = a[live], b[live]
    a, b = kv4.quantise(v)
    vc[slots[live]], vs[slots[live]] = a[live], b[live]
    for p in range(P):
        rows = slice(p * 64, p * 64 + 64)
        for h in range(H):
            assert torch.equal(c.pages[p, h].cpu(), kv4.pack_page(kc[rows, h], ks[rows, h], vc[rows, h], vs[rows, h]))
            want, unit = kv4.bounds(kv4.values(kc[rows, h], ks[rows, h]))
            assert torch.equal(c.bounds[p, h].cpu(), want) and float(c.unit[p, h]) == unit
    c.check()
    for dt in (torch.bfloat16, torch.float16):
        rk, rv = c.read(slots.to(DEV), dt)
        want_k = torch.where(live[:, None, None], kv4.values(*kv4.quantise(k)), 0.0)
        want_v = torch.where(live[:, None, None], kv4.values(*kv4.quantise(v)), 0.0)
        assert rk.dtype == dt and torch.equal(rk.float().cpu(), want_k) and torch.equal(rv.float().cpu(), want_v)


@pytest.mark.parametrize("exp", [-14, 0, 4])
def test_exponents(KV4Cache, exp):
    g = torch.Generator().manual_seed(1)
    k = (torch.randn(64, 1, 64, generator=g) * 2.0 ** (exp + 5)).to(torch.float16)
    c = KV4Cache(1, 1, 64, device=DEV, k_exp=exp, v_exp=exp)
    slots = torch.arange(64, device=DEV)
    c.append(k.to(DEV), -k.to(DEV), slots)
    rk, rv = c.read(slots, torch.float16)
    want = kv4.values(*kv4.quantise(k, exp), exp)
    assert torch.equal(rk.float().cpu(), want) and torch.equal(rv.float().cpu(), -want)
    b, unit = kv4.bounds(want[:, 0])
    assert torch.equal(c.bounds[0, 0].cpu(), b) and float(c.unit[0, 0]) == unit


def test_strided_and_unaligned_rows(KV4Cache):
    """Slices of a fused projection's output, and rows that do not start on 16 bytes."""
    g = torch.Generator().manual_seed(2)
    H, D, T = 2, 128, 33
    qkv = torch.randn(T, 8, D, generator=g).to(torch.bfloat16).to(DEV)
    odd = torch.randn(T, 2 * H * (D + 1) + 1, generator=g).to(torch.bfloat16).to(DEV)
    slots = torch.arange(T, device=DEV)
    for k, v in ((qkv[:, 4:6], qkv[:, 6:8]),
                 (odd[:, 1:1 + H * (D + 1)].unflatten(1, (H, D + 1))[..., 1:], odd[:, 1:1 + H * (D + 1)].unflatten(1, (H, D + 1))[..., :D])):
        c = KV4Cache(1, H, D, device=DEV)
        c.append(k, v, slots)
        rk, rv = c.read(slots)
        assert torch.equal(rk.float().cpu(), kv4.values(*kv4.quantise(k.cpu())))
        assert torch.equal(rv.float().cpu(), kv4.values(*kv4.quantise(v.cpu())))


def test_status_of_bad_slots_and_values(KV4Cache):
    c = KV4Cache(2, 1, 64, device=DEV)
    x = torch.ones(2, 1, 64, dtype=torch.bfloat16, device=DEV)
    c.append(x, x, torch.tensor([0, 128], device=DEV))
    assert int(c.status) == 1
    with pytest.raises(RuntimeError, match="out of range"):
        c.check()
    c.status.zero_()
    k, v = c.read(torch.tensor([128, 0], device=DEV))
    one = kv4.values(*kv4.quantise(x.cpu()))[0].to(DEV)                 # 1 is held as 6 * 11/64
    assert int(c.status) == 1 and (k[0] == 0).all() and torch.equal(k[1].float(), one)
    c.status.zero_()
    y = x.clone()
    y[0, 0, 3], y[0, 0, 20], y[1, 0, 5] = math.nan, -math.inf, math.inf
    c.append(y, x, torch.tensor([1, 2], device=DEV))
    assert int(c.status) == 4
    k, _ = c.read(torch.tensor([1, 2], device=DEV))
    assert float(k[0, 0, 3]) == 0 and float(k[0, 0, 20]) == -42 and float(k[1, 0, 5]) == 42
    # block 1 of row 0 holds an infinity: its other values vanish beside it; a NaN leaves its block as it was
    assert torch.equal(k[0, 0, :3].float(), one[0, :3]) and (k[0, 0, 32:].float() == one[0, 32:]).all()


def test_bounds_follow_rewritten_rows(KV4Cache):
    """A rejected draft's row is written again: the page's bounds are those of what it holds now."""
    g = torch.Generator().manual_seed(4)
    c = KV4Cache(1, 1, 64, device=DEV)
    k = torch.randn(64, 1, 64, generator=g).to(torch.bfloat16)
    k[63] *= 30
    c.append(k.to(DEV), k.to(DEV), torch.arange(64, device=DEV))
    k[63] /= 64
    c.append(k[63:].to(DEV), k[63:].to(DEV), torch.tensor([63], device=DEV))
    want, unit = kv4.bounds(kv4.values(*kv4.quantise(k))[:, 0])
    assert torch.equal(c.bounds[0, 0].cpu(), want) and float(c.unit[0, 0]) == unit


# ---------------------------------------------------------------------------------- attention
STEP = [
    ([1], [1], 1, 1, 64, torch.bfloat16, 0),
    ([64], [1], 2, 8, 128, torch.bfloat16, 0),
    ([65, 63, 0, 129], [1, 1, 1, 1], 2, 3, 128, torch.float16, 0),
    ([200, 1, 70], [3, 2, 3], 2, 5, 256, torch.bfloat16, 0),          # verify rows; one sequence shorter than its rows
    ([300, 128], [2, 0], 1, 12, 64, torch.float16, 0),                # a sequence without rows
    ([500], [4], 1, 6, 128, torch.bfloat16, 100),                     # window
    ([130, 64], [1, 1], 1, 40, 128, torch.bfloat16, 1),               # more heads than a tile; window of one
    ([777], [1], 4, 16, 256, torch.float16, 300),
    ([900, 40], [3, 3], 1, 7, 128, torch.bfloat16, 0),                # three row groups of eight
    ([3000], [3], 1, 8, 64, torch.bfloat16, 0),                       # and split over blocks
    ([700], [4], 2, 8, 128, torch.float16, 0),
]
PROMPT = [
    ([100], [100], 1, 1, 64, torch.bfloat16, 0),
    ([300, 65, 7, 130], [130, 65, 9, 1], 2, 2, 128, torch.bfloat16, 0),
    ([400], [70], 1, 5, 256, torch.float16, 0),
    ([257, 0], [33, 3], 2, 8, 64, torch.float16, 0),
    ([450], [90], 1, 4, 128, torch.bfloat16, 37),
    ([129], [129], 1, 3, 128, torch.float16, 64),
    ([3000], [60], 1, 2, 64, torch.bfloat16, 0),                      # a tile's keys split over blocks
    ([2100, 1030], [40, 40], 1, 2, 256, torch.bfloat16, 0),
    ([2500], [40], 1, 1, 128, torch.float16, 1100),
]


@pytest.mark.parametrize("lens,news,H,G,D,dtype,window", STEP + PROMPT)
def test_attend(KV4Cache, lens, news, H, G, D, dtype, window):
    x = Batch(lens, news, H, G, D, dtype, seed=sum(lens), q_scale=2.0)
    c = x.cache(KV4Cache)
    scale = D ** -0.5
    out, lse = c.attend(*x.args(), scale, max_q=max(news), window=window, return_lse=True)
    c.check()
    assert out.dtype == dtype
    check(out, lse, x.oracle(scale, window), max(lens))
    again = c.attend(*x.args(), scale, max_q=max(news), window=window)
    assert torch.equal(again, out)                                   # and bit for bit again


@pytest.mark.parametrize("max_q,scale", [(3, 0.3), (200, 0.3), (3, -0.2), (200, -0.2), (3, 0.0), (200, 0.0)])
def test_both_kernels_and_any_scale(KV4Cache, max_q, scale):
    """max_q only chooses the kernel; negative and zero scales."""
    x = Batch([333, 90], [3, 2], 2, 4, 128, seed=9)
    c = x.cache(KV4Cache)
    out, lse = c.attend(*x.args(), scale, max_q=max_q, return_lse=True)
    check(out, lse, x.oracle(scale), 333)


@pytest.mark.parametrize("max_q", [2, 500])
def test_large_and_tiny_queries(KV4Cache, max_q):
    """bf16 rows far outside f16's range, a row of zeros, and scores that move the running maximum late."""
    x = Batch([640], [2], 1, 4, 128, seed=10)
    x.q[0, 0] *= 2.0 ** 60
    x.q[0, 1] *= 2.0 ** -70
    x.q[1, 0] = 0
    x.q[1, 2] *= 40
    x.k[600:] *= 3                                                   # the largest keys come last
    c = x.cache(KV4Cache)
    q, cu, sl, tb = x.args()
    out = c.attend(q, cu, sl, tb, 2.0 ** -3, max_q=max_q)
    o, _, mag = x.oracle(2.0 ** -3)
    rows = [(0, 1), (0, 2), (0, 3), (1, 0), (1, 1), (1, 3)]
    for r, h in rows:
        assert ((out[r, h].double().cpu() - o[r, h]).abs() <= 2.0 ** -8 * o[r, h].abs() + 2.0 ** -9 * mag[r, h] + 1e-6).all()
    # scores of 2^60: one key takes all (its f32 score is the largest)
    assert torch.isfinite(out).all()


def test_unwritten_bytes_may_be_anything(KV4Cache):
    """NaN scales in positions that no row sees, in both kernels and over chosen pages."""
    x = Batch([70, 1], [2, 1], 1, 4, 128, seed=11)
    c = x.cache(KV4Cache)
    ref = c.attend(*x.args(), 0.1, max_q=2)
    k, v = (t.to(DEV) for t in (x.k, x.v))
    c.pages.fill_(0xFF)
    c.append(k, v, x.slots.to(DEV))
    for max_q in (2, 100):
        assert torch.allclose(c.attend(*x.args(), 0.1, max_q=max_q).float(), ref.float(), atol=2e-2)
        assert torch.isfinite(c.attend(*x.args(), 0.1, max_q=max_q)).all()
    pages = torch.tensor([[[1, 0]], [[0, 1]], [[0, -1]]], dtype=torch.int32, device=DEV)
    assert torch.equal(c.attend(*x.args(), 0.1, max_q=2, pages=pages), ref) or torch.allclose(
        c.attend(*x.args(), 0.1, max_q=2, pages=pages).float(), ref.float(), atol=2e-2)


def test_a_bad_row_stays_its_own(KV4Cache):
    x = Batch([100], [3], 1, 4, 64, seed=12)
    c = x.cache(KV4Cache)
    ref = {m: c.attend(*x.args(), 0.1, max_q=m) for m in (3, 100)}
    x.q[1, 2, 5] = math.nan
    for m in (3, 100):
        out = c.attend(*x.args(), 0.1, max_q=m)
        assert torch.isnan(out[1, 2]).all()
        out[1, 2], ref[m][1, 2] = 0, 0
        assert torch.equal(out, ref[m])


@pytest.mark.parametrize("lens,news,H,G,D,dtype", [
    ([640, 65, 30], [1, 2, 1], 2, 8, 128, torch.bfloat16), ([900], [40], 1, 3, 64, torch.float16),
    ([520, 1], [2, 3], 2, 20, 256, torch.bfloat16)])
def test_attend_over_chosen_pages(KV4Cache, lens, news, H, G, D, dtype):
    x = Batch(lens, news, H, G, D, dtype, seed=13)
    c = x.cache(KV4Cache)
    g = torch.Generator().manual_seed(1)
    T = sum(news)
    pages = torch.full((T, H, 5), -1, dtype=torch.int32)
    for r in range(T):
        for h in range(H):
            some = torch.randperm(max(1, max(lens) // 64), generator=g)[:5].int()   # in any order, past the end too
            pages[r, h, :some.numel()] = some
    pages[0, 0] = -1                                                  # a row without pages
    out, lse = c.attend(*x.args(), 0.09, max_q=max(news), pages=pages.to(DEV), return_lse=True)
    for r in range(T):                                                # what lies past a row's own position is not seen
        b = int(torch.searchsorted(x.cu, torch.tensor(r, dtype=torch.int32), right=True)) - 1
        p = lens[b] - news[b] + r - int(x.cu[b])
        pages[r][pages[r] * 64 > p] = -1
    check(out, lse, x.oracle(0.09, pages=pages), 320)


@pytest.mark.parametrize("D,T,n", [(128, 1024, 6000), (64, 700, 5000), (256, 600, 4000)])
def test_long_prompts_are_whole_and_the_same_every_time(KV4Cache, D, T, n):
    """Every row of many tiles, some whole and some with their keys split, against f32 on the GPU, over and over:
    an output read before its last products shows in some rows of some runs."""
    H, G = 8, 4
    g = torch.Generator(device=DEV).manual_seed(D)
    k = (torch.randn(n, H, D, generator=g, device=DEV) * 1.3 + 0.3).bfloat16()
    v = torch.randn(n, H, D, generator=g, device=DEV).bfloat16()
    q = (torch.randn(T, H * G, D, generator=g, device=DEV) * 1.5).bfloat16()
    pages = -(-n // 64)
    c = KV4Cache(pages, H, D, device=DEV)
    table = torch.randperm(pages, generator=g, device=DEV).int()[None]
    j = torch.arange(n, device=DEV)
    slots = table[0, j // 64].long() * 64 + j % 64
    c.append(k, v, slots)
    hk, hv = (x.float() for x in c.read(slots))
    s = torch.einsum("thgd,nhd->htgn", q.float().unflatten(1, (H, G)), hk) * D ** -0.5
    s.masked_fill_((j > torch.arange(n - T, n, device=DEV)[:, None])[None, :, None], -math.inf)
    want = torch.einsum("htgn,nhd->thgd", torch.softmax(s, -1), hv).flatten(1, 2)
    cu = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    first = c.attend(q, cu, lens, table, D ** -0.5)
    assert float((first.float() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max()) + 2.0 ** -9
    for _ in range(30):
        assert torch.equal(c.attend(q, cu, lens, table, D ** -0.5), first)
    c.check()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_rows_that_fall_behind(KV4Cache, D):
    """The rows of one warp in four see scores that rise without end (their outputs are rescaled again and again),
    the other rows see equal scores: the slow warp's neighbours may be a whole step ahead of it."""
    H, G, T, n = 8, 4, 512, 6000
    g = torch.Generator(device=DEV).manual_seed(D)
    j = torch.arange(n, device=DEV)
    ramp = 3.0 * (j + 64) / n
    k = (ramp[:, None] * (1 + torch.arange(D, device=DEV) // 16 / 16.0)).bfloat16()[:, None].expand(n, H, D)
    v = torch.randn(n, H, D, generator=g, device=DEV).bfloat16()
    sign = 1.0 - 2.0 * (torch.arange(D, device=DEV) % 2)
    steep = (torch.arange(T, device=DEV) // 8 % 4 == 1)[:, None]         # 8 tokens x 4 rows: a warp's rows
    q = torch.where(steep, torch.full_like(sign, 2048.0 / D), sign).bfloat16()[:, None].expand(T, H * G, D)
    pages = -(-n // 64)
    c = KV4Cache(pages, H, D, device=DEV)
    table = torch.randperm(pages, generator=g, device=DEV).int()[None]
    slots = table[0, j // 64].long() * 64 + j % 64
    c.append(k, v, slots)
    hk, hv = (x.double() for x in c.read(slots))
    scale = 1.0 / 8
    want = torch.empty(T, H * G, D, dtype=torch.float64, device=DEV)
    for h in range(H):
        s = torch.einsum("tgd,nd->tgn", q[:, h * G:(h + 1) * G].double(), hk[:, h]) * scale
        s.masked_fill_((j > torch.arange(n - T, n, device=DEV)[:, None])[:, None], -math.inf)
        want[:, h * G:(h + 1) * G] = torch.softmax(s, -1) @ hv[:, h]
    cu = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    first = c.attend(q, cu, lens, table, scale)
    # half an ulp of bf16, P in f16, and exp2 of differences between scores (sums of few-bit values: exact) near 2^11
    assert float((first.double() - want).abs().max()) <= (2.0 ** -9 + 2.0 ** -10 + 2.0 ** -11) * float(hv.abs().max())
    for _ in range(30):
        assert torch.equal(c.attend(q, cu, lens, table, scale), first)
    c.check()


def test_many_sequences(KV4Cache):
    """More sequences than threads of a block, most of them short, tiles split over blocks."""
    g = torch.Generator().manual_seed(14)
    lens = [int(x) for x in torch.randint(0, 40, (300,), generator=g)]
    lens[7], lens[250] = 1500, 900
    x = Batch(lens, [1] * 300, 1, 2, 64, seed=15)
    c = x.cache(KV4Cache)
    out, lse = c.attend(*x.args(), 0.2, max_q=1, return_lse=True)
    check(out, lse, x.oracle(0.2), 1500)


def test_offsets_past_32_bits(KV4Cache):
    """A pool of 5 GB: the last pages are written, read and attended to."""
    H, D = 8, 256
    P = 5 * 2 ** 30 // (H * 72 * D)
    c = KV4Cache(P, H, D, device=DEV)
    g = torch.Generator().manual_seed(16)
    k = torch.randn(80, H, D, generator=g).to(torch.bfloat16)
    table = torch.tensor([[P - 1, P - 2]], dtype=torch.int32)
    j = torch.arange(80)
    slots = table[0, j // 64].long() * 64 + j % 64
    c.append(k.to(DEV), k.to(DEV), slots.to(DEV))
    rk, _ = c.read(slots.to(DEV))
    held = kv4.values(*kv4.quantise(k))
    assert torch.equal(rk.float().cpu(), held)
    q = torch.randn(1, H, D, generator=g).to(torch.bfloat16)
    s = torch.einsum("hd,nhd->hn", q[0].double(), held.double()) * 0.06
    want = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), held.double())
    for max_q in (1, 100):
        out = c.attend(q.to(DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV),
                       torch.tensor([80], dtype=torch.int32, device=DEV), table.to(DEV), 0.06, max_q=max_q)
        assert (out[0].double().cpu() - want).abs().max() <= 2.0 ** -8 * want.abs().max()
    del c
    torch.cuda.empty_cache()


def test_bad_page_is_skipped_and_reported(KV4Cache):
    x = Batch([200], [1], 1, 2, 64, seed=17)
    for max_q in (1, 200):
        c = x.cache(KV4Cache)
        q, cu, sl, tb = x.args()
        bad = tb.clone()
        bad[0, 1] = x.n_pages
        c.attend(q, cu, sl, bad, 0.1, max_q=max_q)
        assert int(c.status) == 1
    c = x.cache(KV4Cache)
    c.attend(q, cu, sl, tb, 0.1, pages=torch.tensor([[[0, 9]]], dtype=torch.int32, device=DEV))
    assert int(c.status) == 1


def test_queries_in_any_layout(KV4Cache):
    x = Batch([150], [2], 2, 4, 128, seed=18)
    c = x.cache(KV4Cache)
    q, cu, sl, tb = x.args()
    ref = c.attend(q, cu, sl, tb, 0.1, max_q=2)
    wide = torch.zeros(2, 8 + 4, 128, dtype=q.dtype, device=DEV)
    wide[:, 2:10] = q
    assert torch.equal(c.attend(wide[:, 2:10], cu, sl, tb, 0.1, max_q=2), ref)
    odd = torch.zeros(2 * 8 * 129 + 1, dtype=q.dtype, device=DEV)[1:].view(2, 8, 129)
    odd[..., :128] = q
    assert torch.equal(c.attend(odd[..., :128], cu, sl, tb, 0.1, max_q=2), ref)
    t = q.transpose(1, 2).contiguous().transpose(1, 2)               # inner stride not 1
    assert torch.equal(c.attend(t, cu, sl, tb, 0.1, max_q=2), ref)


# ---------------------------------------------------------------------------- choosing pages
def choose(x, budget, first, last):
    """The definition: exact scores in 64 bits, ties to the lowest page."""
    T = x.q.shape[0]
    pages = torch.full((T, x.H, budget), -1, dtype=torch.int32)
    held, at = x.held(x.k), 0
    for b, (n, m) in enumerate(zip(x.lens, x.news)):
        w = -(-n // 64)
        k = torch.cat([held[at:at + n], torch.zeros(w * 64 - n, x.H, x.D, dtype=torch.float64)]).view(w, 64, x.H, x.D)
        bnd = [[kv4.bounds(k[i, :, h]) for h in range(x.H)] for i in range(w)]
        at += n
        for i in range(m):
            row, p = int(x.cu[b]) + i, n - m + i
            if p < 0:
                continue
            cnt = p // 64 + 1
            for h in range(x.H):
                if cnt <= budget:
                    pages[row, h, :cnt] = torch.arange(cnt)
                    continue
                q = torch.nan_to_num(x.q[row, h * x.G:(h + 1) * x.G].double(), nan=0.0, posinf=3.4028235e38, neginf=-3.4028235e38)
                f = torch.tensor([kv4.bounds(y[None])[1] for y in q])
                r = torch.round(q / f[:, None])
                score = []
                for page in range(first, cnt - last):
                    e, unit = bnd[page][h]
                    s = r.clamp(min=0) @ e[0].double() + r.clamp(max=0) @ e[1].double()
                    score.append((-float((s * f).max()) * unit, page))
                best = [pg for _, pg in sorted(score)[:budget - first - last]]
                chosen = list(range(first)) + sorted(best) + list(range(cnt - last, cnt))
                pages[row, h] = torch.tensor(chosen)
    return pages


@pytest.mark.parametrize("lens,news,H,G,D,dtype,budget,first,last", [
    ([1000, 64, 0, 700], [1, 1, 1, 1], 2, 8, 128, torch.bfloat16, 6, 1, 2),
    ([900, 30], [3, 2], 1, 1, 64, torch.float16, 4, 0, 1),
    ([700], [70], 2, 2, 64, torch.bfloat16, 5, 1, 1),
    ([650], [9], 1, 4, 256, torch.float16, 3, 1, 2),                  # nothing left to compete for
    ([800, 400], [2, 17], 1, 5, 128, torch.bfloat16, 7, 2, 2),
    ([640], [1], 1, 12, 128, torch.bfloat16, 5, 1, 2),
    ([640], [2], 1, 64, 64, torch.float16, 5, 1, 2),
    ([700], [3], 3, 3, 128, torch.bfloat16, 20, 1, 2),                # budget larger than the pages
])
def test_select(KV4Cache, lens, news, H, G, D, dtype, budget, first, last):
    x = Batch(lens, news, H, G, D, dtype, seed=budget + sum(lens))
    c = x.cache(KV4Cache)
    got = c.select(*x.args(), budget, first=first, last=last, max_q=max(news))
    c.check()
    assert torch.equal(got.cpu(), choose(x, budget, first, last))


def test_select_ties_go_to_the_lowest_page(KV4Cache):
    x = Batch([64 * 12], [1], 1, 2, 64, seed=20)
    x.k[:] = x.k[:1]                                                  # every page the same
    c = x.cache(KV4Cache)
    assert c.select(*x.args(), 6)[0, 0].tolist() == [0, 1, 2, 3, 10, 11]
    x.q[:] = 0                                                        # every score zero
    assert c.select(*x.args(), 6)[0, 0].tolist() == [0, 1, 2, 3, 10, 11]
    x.q[0, 0, 0], x.q[0, 1, 3] = math.nan, math.inf
    got = c.select(*x.args(), 6)
    assert torch.equal(got.cpu(), choose(x, 6, 1, 2))


@pytest.mark.parametrize("width", [250, 500, 1000, 1100, 5000])
def test_select_of_long_rows(KV4Cache, width):
    """Each way of finding the threshold, on bounds that are set directly: with ties, in every width."""
    g = torch.Generator().manual_seed(width)
    c = KV4Cache(width, 1, 64, device=DEV)
    c.bounds.copy_(torch.randint(-3, 4, c.bounds.shape, generator=g).to(torch.int8))
    c.unit.copy_(2.0 ** torch.randint(-2, 3, c.unit.shape, generator=g).float())
    q = torch.zeros(3, 1, 64, dtype=torch.bfloat16)
    q[0, 0, 5], q[1, 0, :3], q[2] = 1, torch.tensor([1.0, -1.0, 0.5]), torch.randn(1, 64, generator=g).bfloat16()
    table = torch.randperm(width, generator=g).int()[None]
    cu = torch.tensor([0, 3], dtype=torch.int32)
    sl = torch.tensor([width * 64], dtype=torch.int32)
    for budget in (4, 33, width - 1):
        got = c.select(q.to(DEV), cu.to(DEV), sl.to(DEV), table.to(DEV), budget).cpu()
        b, u = c.bounds.cpu()[table[0].long(), 0].double(), c.unit.cpu()[table[0].long(), 0].double()
        for r in range(3):
            f = kv4.bounds(q[r].double())[1]
            y = torch.round(q[r, 0].double() / f)
            s = (b[:, 0] @ y.clamp(min=0) + b[:, 1] @ y.clamp(max=0)) * f * u
            order = sorted(range(1, width - 2), key=lambda i: (-float(s[i]), i))[:budget - 3]
            assert got[r, 0].tolist() == [0] + sorted(order) + [width - 2, width - 1]


@pytest.mark.parametrize("width", [500, 600, 1000])
def test_select_of_many_rows_is_the_choice_of_each(KV4Cache, width):
    """Many rows at once and a few at a time are chosen for in different ways: the choices are the same, ties too."""
    g = torch.Generator().manual_seed(width)
    T, H, D, n = 160, 2, 64, 400
    c = KV4Cache(n, H, D, device=DEV)
    c.bounds.copy_(torch.randint(-3, 4, c.bounds.shape, generator=g).to(torch.int8))
    c.unit.copy_(2.0 ** torch.randint(-2, 3, c.unit.shape, generator=g).float())
    q = torch.randn(T, H * 2, D, generator=g).bfloat16()
    q[::3] = torch.round(q[::3])                                      # with ties
    table = torch.randint(0, n, (T, width), generator=g).int().to(DEV)
    sl = torch.randint(width * 32, width * 64 + 1, (T,), generator=g).int().to(DEV)
    q, cu = q.to(DEV), torch.arange(T + 1).int().to(DEV)
    for budget in (5, 64, 300):
        all_rows = c.select(q, cu, sl, table, budget, max_q=1)
        for i in range(0, T, 20):
            part = c.select(q[i:i + 20], cu[:21], sl[i:i + 20], table[i:i + 20], budget, max_q=1)
            assert torch.equal(part, all_rows[i:i + 20])
    c.check()


def test_chosen_pages_hold_the_best_key(KV4Cache):
    """The score is an upper bound: a page with a key far above the others is always taken."""
    x = Batch([64 * 40], [1], 2, 4, 128, seed=21)
    c0 = x.k.clone()
    x.k = (c0 * 0.1).to(x.dtype)
    q = x.q[0].view(2, 4, 128)
    for h in range(2):
        x.k[64 * 17 + 5, h] = (q[h, 2] * 4).to(x.dtype)
    c = x.cache(KV4Cache)
    got = c.select(*x.args(), 8)
    assert all(17 in got[0, h].tolist() for h in range(2))


# ------------------------------------------------------------------------ streams, graphs, refusals
def test_other_stream_and_graph(KV4Cache):
    x = Batch([700, 300], [1, 1], 2, 8, 128, seed=22)
    c = x.cache(KV4Cache)
    args = x.args()
    ref_pages = c.select(*args, 5, max_q=1)
    ref = c.attend(*args, 0.1, max_q=1, pages=ref_pages)
    full = c.attend(*args, 0.1, max_q=1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        pages = c.select(*args, 5, max_q=1)
        out = c.attend(*args, 0.1, max_q=1, pages=pages)
    s.synchronize()
    assert torch.equal(pages, ref_pages) and torch.equal(out, ref)
    g = torch.cuda.CUDAGraph()
    slots = torch.zeros(2, dtype=torch.int64, device=DEV)
    kn, vn = (torch.zeros(2, 2, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    slots.fill_(-1)
    with torch.cuda.graph(g):
        c.append(kn, vn, slots)
        pages = c.select(*args, 5, max_q=1)
        out = c.attend(*args, 0.1, max_q=1, pages=pages)
        whole = c.attend(*args, 0.1, max_q=1)
    for _ in range(3):
        out.zero_(), whole.zero_(), pages.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(pages, ref_pages) and torch.equal(out, ref) and torch.equal(whole, full)
    c.check()


def test_empty_calls(KV4Cache):
    x = Batch([10], [0], 1, 2, 64, seed=23)
    c = x.cache(KV4Cache)
    out, lse = c.attend(*x.args(), 0.1, return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    assert c.select(*x.args(), 4).shape == (0, 1, 4)
    e = torch.zeros(0, 1, 64, dtype=torch.bfloat16, device=DEV)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    c.append(e, e, none)
    assert c.read(none)[0].shape == (0, 1, 64)


def test_refusals(KV4Cache):
    x = Batch([100], [2], 2, 2, 64, seed=24)
    c = x.cache(KV4Cache)
    q, cu, sl, tb = x.args()
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=DEV)
    s = torch.arange(3, device=DEV)
    bad = [
        lambda: c.append(k, k, s.int()),
        lambda: c.append(k, k, s[:2]),
        lambda: c.append(k.float(), k.float(), s),
        lambda: c.append(k, k.half(), s),
        lambda: c.append(k.cpu(), k, s),
        lambda: c.append(k[:, :1], k, s),
        lambda: c.append(k.transpose(1, 2).contiguous().transpose(1, 2), k, s),
        lambda: c.read(s, torch.float32),
        lambda: c.read(s.cpu()),
        lambda: c.attend(q.float(), cu, sl, tb, 1.0),
        lambda: c.attend(q[:, :3], cu, sl, tb, 1.0),
        lambda: c.attend(q[..., :32], cu, sl, tb, 1.0),
        lambda: c.attend(q, cu.long(), sl, tb, 1.0),
        lambda: c.attend(q, cu[:1], sl, tb, 1.0),
        lambda: c.attend(q, cu, sl.cpu(), tb, 1.0),
        lambda: c.attend(q, cu, sl, tb[0], 1.0),
        lambda: c.attend(q, cu, sl, tb.long(), 1.0),
        lambda: c.attend(q, cu, sl, tb, 1.0, max_q=0),
        lambda: c.attend(q, cu, sl, tb, 1.0, window=-1),
        lambda: c.attend(q, cu, sl, tb, 1.0, pages=torch.zeros(2, 2, 3, device=DEV)),
        lambda: c.attend(q, cu, sl, tb, 1.0, pages=torch.zeros(2, 1, 3, dtype=torch.int32, device=DEV)),
        lambda: c.select(q, cu, sl, tb, 2),
        lambda: c.select(q, cu, sl, tb, 4, last=0),
        lambda: c.select(q, cu, sl, tb, 4, first=-1),
        lambda: c.select(torch.zeros(2, 2 * 65, 64, dtype=q.dtype, device=DEV), cu, sl, tb, 4),
        lambda: c.attend(q, torch.zeros(4098, dtype=torch.int32, device=DEV), torch.zeros(4097, dtype=torch.int32, device=DEV),
                         torch.zeros(4097, 1, dtype=torch.int32, device=DEV), 1.0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            call()
            pytest.fail(f"call {i} was not refused")
    c.check()
    assert torch.isfinite(c.attend(q, cu, sl, tb, 0.1)).all()        # and the cache still works


def test_demo_layer_from_prompt_to_decode():
    """The draft layer of `tools.kv4_demo`: 4-bit keys and values cost what they cost (two e2m1 roundings of
    about 2^-3.3 relative each, averaged over thousands of positions), choosing all pages changes nothing."""
    from vllm_moet_b200.tools.kv4_demo import run
    got = run(hidden=512, heads=8, kv_heads=2, head_dim=64, streams=2, prompt=700, chunk=256, tokens=6, budget=64, sink=None)
    assert got["bytes_per_position"] * 32 == got["bf16_bytes_per_position"] * 9
    assert got["all_pages_rel_err"] < 0.2
    assert abs(got["chosen_pages_rel_err"] - got["all_pages_rel_err"]) < 2e-3      # 64 pages hold every position


# --------------------------------------------------------------------- units that carry no page
@pytest.mark.parametrize("G,D", [(4, 128), (12, 64), (5, 256)])
def test_pages_between_empty_places(KV4Cache, G, D):
    """Choices with a page in every third place: a warp passes over the empty ones, whose ring slots are taken again
    at once.  The same as the choice without gaps up to rounding, and the same bits every time."""
    H, n, m = 2, 2000, 3
    x = Batch([n], [m], H, G, D, seed=31)
    c = x.cache(KV4Cache)
    some = torch.arange(0, 30, 2, dtype=torch.int32)
    gaps = torch.full((m, H, 3 * some.numel()), -1, dtype=torch.int32)
    gaps[..., 1::3] = some
    gaps = gaps.to(DEV)
    out, lse = c.attend(*x.args(), 0.1, max_q=m, pages=gaps, return_lse=True)
    check(out, lse, x.oracle(0.1, pages=gaps.cpu()), 64 * some.numel())
    for _ in range(100):
        again, l2 = c.attend(*x.args(), 0.1, max_q=m, pages=gaps, return_lse=True)
        assert torch.equal(again, out) and torch.equal(l2, lse)
    c.check()


# --------------------------------------------------------------------------- waits that run out
@pytest.mark.parametrize("G,D,pages", [(4, 128, False), (12, 64, True), (5, 256, False), (2, 256, True)])
def test_a_wait_that_runs_out_is_reported(KV4Cache, G, D, pages):
    """A copy that does not come in time (no try is made): the call ends with a status, and what was in flight has
    landed before the block leaves, so the calls after it are whole."""
    x = Batch([3000, 70], [2, 1], 2, G, D, seed=32)
    c = x.cache(KV4Cache)
    chosen = c.select(*x.args(), 9, max_q=2) if pages else None
    ref = c.attend(*x.args(), 0.1, max_q=2, pages=chosen)
    c.check()
    for _ in range(5):
        c._tries = 0
        c.attend(*x.args(), 0.1, max_q=2, pages=chosen)
        assert int(c.status) == 2
        with pytest.raises(RuntimeError, match="wait"):
            c.check()
        c.status.zero_()
        c._tries = KV4Cache._tries
        assert torch.equal(c.attend(*x.args(), 0.1, max_q=2, pages=chosen), ref)
        c.check()


@pytest.mark.parametrize("tries", [1, 2])
def test_a_warp_gives_up_as_one(KV4Cache, tries):
    """Waits that end about when the copy comes: lanes may see either, the warp takes one answer.  The call ends, and it
    is whole or has set the status."""
    x = Batch([2500, 900], [1, 1], 2, 8, 128, seed=33)
    c = x.cache(KV4Cache)
    ref = c.attend(*x.args(), 0.1, max_q=1)
    for _ in range(20):
        c._tries = tries
        out = c.attend(*x.args(), 0.1, max_q=1)
        assert int(c.status) in (0, 2)
        if int(c.status) == 0:
            assert torch.equal(out, ref)
        c.status.zero_()
        c._tries = KV4Cache._tries
        assert torch.equal(c.attend(*x.args(), 0.1, max_q=1), ref)
    c.check()


@pytest.mark.parametrize("D,G,new", [(64, 8, 40), (128, 4, 200), (256, 2, 90)])
def test_a_wait_that_runs_out_in_a_prompt(KV4Cache, D, G, new):
    """The prompt kernel built with short waits: it gives up with products in flight, reports it, and none of them is
    left when the block gives its tensor memory back, so the calls after it are whole."""
    import moet_testkit       # test-only extension (tests/csrc)
    x = Batch([4000, 300], [new, new], 2, G, D, seed=34)
    c = x.cache(KV4Cache)
    args = x.args()
    ref = c.attend(*args, 0.1, max_q=new)
    c.check()
    for _ in range(5):
        moet_testkit.kv4_prompt_wait_test(*args, c.pages, new, torch.empty_like(ref), c.status)
        assert int(c.status) == 2
        c.status.zero_()
        assert torch.equal(c.attend(*args, 0.1, max_q=new), ref)
        c.check()


# ------------------------------------------------------------- pages that are not there, both kernels
@pytest.mark.parametrize("entry", [-1, -7, None, 2 ** 31 - 1])             # None: one past the pool
@pytest.mark.parametrize("lens,news,H,G,D,dtype,window,bad", [
    ([300, 90], [2, 1], 2, 4, 128, torch.float16, 0, 1),
    ([300, 90], [40, 30], 1, 2, 128, torch.bfloat16, 0, 2),
    ([200], [70], 2, 2, 256, torch.float16, 0, 0),
    ([2500], [60], 1, 2, 64, torch.float16, 0, 17),                        # a tile's keys split over blocks
    ([640], [3], 1, 5, 64, torch.bfloat16, 200, 8),
    ([640], [70], 1, 3, 128, torch.float16, 200, 7),
])
def test_a_bad_page_is_left_out_by_both_kernels(KV4Cache, lens, news, H, G, D, dtype, window, bad, entry):
    x = Batch(lens, news, H, G, D, dtype, seed=41)
    c = x.cache(KV4Cache)
    q, cu, sl, tb = x.args()
    tb[0, bad] = x.n_pages if entry is None else entry
    seen = torch.arange(-(-max(lens) // 64), dtype=torch.int32).expand(sum(news), H, -1).clone()
    seen[:news[0]][seen[:news[0]] == bad] = -1
    want = x.oracle(0.1, window, seen)
    for max_q in (max(news), 40 * max(news)):
        out, lse = c.attend(q, cu, sl, tb, 0.1, max_q=max_q, window=window, return_lse=True)
        assert int(c.status) == 1
        c.status.zero_()
        check(out, lse, want, max(lens))


@pytest.mark.parametrize("max_q", [3, 200])
def test_pages_before_the_window_may_be_gone(KV4Cache, max_q):
    """A sliding window's pages are given back as the window leaves them: what no row sees is not looked at."""
    x = Batch([900], [3], 1, 4, 128, seed=42)
    c = x.cache(KV4Cache)
    q, cu, sl, tb = x.args()
    want = x.oracle(0.1, 150)
    first = (900 - 3 - 150 + 1) // 64                                      # 748: page 11
    tb[0, :first] = torch.tensor([-1, -9, x.n_pages, 2 ** 31 - 1] * 3, dtype=torch.int32, device=DEV)[:first]
    out, lse = c.attend(q, cu, sl, tb, 0.1, max_q=max_q, window=150, return_lse=True)
    c.check()
    check(out, lse, want, 900)


# ------------------------------------------------------------------- lengths out of range
@pytest.mark.parametrize("length", [64 * 12 + 1, 2 ** 31 - 1, -1, -2 ** 31])
@pytest.mark.parametrize("max_q", [3, 200])
def test_a_length_out_of_range_is_reported(KV4Cache, length, max_q):
    """More positions than the table holds, or fewer than none; the other sequences are what they were."""
    x = Batch([700, 150, 400], [3, 2, 3], 2, 4, 128, seed=50, width=12)
    c = x.cache(KV4Cache)
    q, cu, sl, tb = x.args()
    tb.clamp_(min=0)
    ref = c.attend(q, cu, sl, tb, 0.1, max_q=max_q)
    ref_pages = c.select(q, cu, sl, tb, 4, max_q=max_q)
    ref_chosen = c.attend(q, cu, sl, tb, 0.1, max_q=max_q, pages=ref_pages)
    c.check()
    sl[1] = length
    rest = [0, 1, 2, 5, 6, 7]
    for call, want in ((lambda: c.attend(q, cu, sl, tb, 0.1, max_q=max_q), ref),
                       (lambda: c.attend(q, cu, sl, tb, 0.1, max_q=max_q, window=300), None),
                       (lambda: c.select(q, cu, sl, tb, 4, max_q=max_q), ref_pages),
                       (lambda: c.select(q, cu, sl, tb, 12, max_q=max_q), None),
                       (lambda: c.attend(q, cu, sl, tb, 0.1, max_q=max_q, pages=ref_pages), ref_chosen)):
        got = call()
        assert int(c.status) == 1
        c.status.zero_()
        if want is not None:
            got, want = got[rest].float(), want[rest].float()
            assert torch.allclose(got, want, rtol=2.0 ** -7, atol=2.0 ** -9 * 6)      # split elsewhere: a rounding apart


# ------------------------------------------------------------------------ row offsets out of range
@pytest.mark.parametrize("cu", [[0, 3, 9, 8], [-1, 3, 5, 8], [0, 5, 3, 8]])
@pytest.mark.parametrize("max_q", [8, 200])
def test_offsets_out_of_range_are_reported(KV4Cache, cu, max_q):
    x = Batch([700, 150, 400], [3, 2, 3], 2, 4, 128, seed=51)
    c = x.cache(KV4Cache)
    q, _, sl, tb = x.args()
    tb.clamp_(min=0)
    cu = torch.tensor(cu, dtype=torch.int32, device=DEV)
    pages = torch.zeros(8, 2, 3, dtype=torch.int32, device=DEV)
    for call in (lambda: c.attend(q, cu, sl, tb, 0.1, max_q=max_q), lambda: c.attend(q, cu, sl, tb, 0.1, max_q=max_q, pages=pages),
                 lambda: c.select(q, cu, sl, tb, 4, max_q=max_q), lambda: c.select(q, cu, sl, tb, 400, max_q=max_q)):
        call()
        assert int(c.status) == 1
        c.status.zero_()


# -------------------------------------------------------------------- rows that belong to no sequence
def poison(*shapes):
    """NaN into the blocks that the allocator gives out next for these sizes."""
    x = [torch.full(s, math.nan, dtype=d, device=DEV) for s, d in shapes for _ in range(3)]
    torch.cuda.synchronize()
    del x


@pytest.mark.parametrize("before,after", [(0, 3), (2, 0), (5, 700)])
@pytest.mark.parametrize("news,max_q,G,D,dtype", [([2, 1], 2, 4, 128, torch.float16), ([2, 1], 400, 4, 128, torch.bfloat16),
                                                  ([50, 3], 50, 2, 64, torch.float16), ([3, 70], 70, 3, 256, torch.bfloat16)])
def test_rows_of_no_sequence_are_zeros(KV4Cache, news, max_q, G, D, dtype, before, after):
    """A batch padded to a captured size: rows in front of cu_q[0] and past cu_q[B]."""
    H = 2
    x = Batch([700, 64 * 9], news, H, G, D, dtype, seed=43)
    c = x.cache(KV4Cache)
    q, cu, sl, tb = x.args()
    n = sum(news)
    wide = torch.randn(before + n + after, H * G, D, device=DEV).to(dtype)
    wide[before:before + n] = q
    cu = cu + before
    ref_pages = c.select(q, cu - before, sl, tb, 5, max_q=max_q)
    for chosen in (False, True):
        pages = None
        if chosen:
            pages = c.select(wide, cu, sl, tb, 5, max_q=max_q)
            assert torch.equal(pages[before:before + n], ref_pages)
            assert (pages[:before] == -1).all() and (pages[before + n:] == -1).all()
            pages[:before], pages[before + n:] = ref_pages[0], ref_pages[0]          # and whatever they ask for
        want = x.oracle(0.1, pages=ref_pages.cpu() if chosen else None)
        poison((wide.shape, dtype), (wide.shape[:2], torch.float32))
        out, lse = c.attend(wide, cu, sl, tb, 0.1, max_q=max_q, pages=pages, return_lse=True)
        check(out[before:before + n], lse[before:before + n], want, 700)
        assert (out[:before] == 0).all() and (out[before + n:] == 0).all()
        assert (lse[:before] == -math.inf).all() and (lse[before + n:] == -math.inf).all()
    c.check()


@pytest.mark.parametrize("max_q", [1, 100])
def test_a_batch_without_sequence_rows(KV4Cache, max_q):
    x = Batch([100, 0], [0, 0], 1, 2, 64, seed=44)
    c = x.cache(KV4Cache)
    _, cu, sl, tb = x.args()
    q = torch.randn(5, 2, 64, device=DEV).bfloat16()
    poison((q.shape, q.dtype), (q.shape[:2], torch.float32))
    out, lse = c.attend(q, cu, sl, tb, 0.1, max_q=max_q, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert (c.select(q, cu, sl, tb, 3, max_q=max_q) == -1).all()
    c.check()


# ----------------------------------------------------------------------------- max_q below the rows
@pytest.mark.parametrize("news,max_q,G,D", [([200, 9], 40, 8, 128), ([90, 200], 64, 4, 64), ([200, 20], 33, 2, 256)])
def test_more_rows_than_max_q_are_reported(KV4Cache, news, max_q, G, D):
    """The rows up to max_q are whole; those past it are zeros (no pages), and the status says so."""
    x = Batch([900, 700], news, 2, G, D, seed=45)
    c = x.cache(KV4Cache)
    args = x.args()
    ref, ref_lse = c.attend(*args, 0.1, max_q=max(news), return_lse=True)
    ref_pages = c.select(*args, 5, max_q=max(news))
    c.check()
    some = torch.cat([torch.arange(n) < max_q for n in news]).to(DEV)
    poison((ref.shape, ref.dtype), (ref.shape[:2], torch.float32))
    out, lse = c.attend(*args, 0.1, max_q=max_q, return_lse=True)
    assert int(c.status) == 3
    c.status.zero_()
    assert torch.isfinite(out).all() and (out[~some] == 0).all() and (lse[~some] == -math.inf).all()
    # another plan may cut a tile's keys elsewhere: P in f16 and one rounding of the output apart
    assert torch.allclose(out[some].float(), ref[some].float(), rtol=2.0 ** -7, atol=2.0 ** -9 * 6)
    assert torch.allclose(lse[some], ref_lse[some], rtol=0, atol=2.0 ** -11)
    pages = c.select(*args, 5, max_q=max_q)
    assert int(c.status) == 3
    assert torch.equal(pages[some], ref_pages[some])
    assert (pages[~some] == -1).all()


# ------------------------------------------------------------------------------------ huge windows
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 64 * 5, 64 * 5 - 1])
@pytest.mark.parametrize("max_q", [20, 200])
def test_a_window_past_the_table_hides_nothing(KV4Cache, window, max_q):
    """With sequences that are shorter than their rows: positions below zero take part in the window's arithmetic."""
    x = Batch([5, 300], [20, 7], 1, 1, 64, seed=46)
    c = x.cache(KV4Cache)
    args = x.args()
    out, lse = c.attend(*args, 0.2, max_q=max_q, window=window, return_lse=True)
    check(out, lse, x.oracle(0.2, window), 300)
    pages = torch.arange(5, dtype=torch.int32, device=DEV).expand(27, 1, 5).contiguous()
    out, lse = c.attend(*args, 0.2, max_q=max_q, window=window, pages=pages, return_lse=True)
    check(out, lse, x.oracle(0.2, window), 300)
    c.check()


# -------------------------------------------------------------------------------- long flat tails
@pytest.mark.parametrize("bits", [25.05, 24.5, 20.3])
@pytest.mark.parametrize("mode", ["step", "prompt", "chosen"])
@pytest.mark.parametrize("D", [64, 256])
def test_small_weights_of_a_long_tail_count(KV4Cache, D, mode, bits):
    """One key takes nearly all; 131071 others weigh 2^-bits of it each.  In f16 beside a weight of 1 they would be
    subnormal or nothing.  Enough rows that a warp has many of a row's pages.  Bound: half an ulp of f16, 2^-11 for a
    weight in f16, 2^-12 for the sum and the exponent; in a prompt the largest weight is held as 2^7 at least, so each
    weight is off by half a subnormal step, 2^-25 / 2^7 of it, at most."""
    n, G, H = 131072, 2, 8
    B, m = (1, 40) if mode == "prompt" else (64, 1)
    k = torch.zeros(n, H, D, dtype=torch.float16, device=DEV)
    v = torch.full((n, H, D), 1.5, dtype=torch.float16, device=DEV)
    k[70], v[70] = 1.5, 0                                             # 1.5 = 6 * 0.25: held as it is
    c = KV4Cache(n // 64, H, D, device=DEV)
    c.append(k, v, torch.arange(n, device=DEV))
    rk, rv = c.read(torch.tensor([70, 71], device=DEV), torch.float16)
    assert (rk[0] == 1.5).all() and (rk[1] == 0).all() and (rv[1] == 1.5).all()
    q = torch.full((B * m, H * G, D), 0.5, dtype=torch.float16, device=DEV)
    scale = bits * math.log(2) / (D * 0.75)
    cu = torch.arange(B + 1, dtype=torch.int32, device=DEV) * m
    sl = torch.full((B,), n, dtype=torch.int32, device=DEV)
    table = torch.arange(n // 64, dtype=torch.int32, device=DEV).expand(B, -1).contiguous()
    pages = table[:, None].expand(B, H, -1).contiguous() if mode == "chosen" else None
    out, lse = c.attend(q, cu, sl, table, scale, max_q=1 if mode != "prompt" else 80, pages=pages, return_lse=True)
    for i in range(B * m):
        tail = (n - m + i % m) * 2.0 ** -bits                         # the positions up to the row's own, less the one
        want = 1.5 * tail / (1 + tail)
        bound = (2.0 ** -11 + 2.0 ** -11 + 2.0 ** -12) * want + (1.5 * n * 2.0 ** -32 if mode == "prompt" else 0)
        assert ((out[i].double() - want).abs() <= bound).all(), (out[i, 0, 0], want)
        assert ((lse[i].double() - (bits * math.log(2) + math.log1p(tail))).abs() <= 2.0 ** -11).all()
    c.check()


# ------------------------------------------------------------------------------- the largest queries
@pytest.mark.parametrize("max_q", [2, 500])
def test_bf16_queries_up_to_the_type_s_largest(KV4Cache, max_q):
    x = Batch([300], [2], 1, 4, 64, seed=48)
    x.k = (x.k.float() * 2.0 ** -6).to(torch.bfloat16)
    x.q[0, 1] = (x.q[0, 1].float() * 2.0 ** 124).clamp(-3.38e38, 3.38e38).to(torch.bfloat16)
    x.q[1, 3, ::2] = -3.3895314e38                                     # the type's lowest value
    x.q[1, 3, 1::2] = 3.3895314e38
    assert torch.isfinite(x.q).all()
    c = x.cache(KV4Cache)
    scale = 2.0 ** -121
    out, lse = c.attend(*x.args(), scale, max_q=max_q, return_lse=True)
    check(out, lse, x.oracle(scale), 300)


# --------------------------------------------------------------------------------- negative zeros
@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_negative_zeros_keep_their_sign(KV4Cache, D, dtype):
    g = torch.Generator().manual_seed(49)
    k = torch.randn(64, 1, D, generator=g).to(dtype)
    k[:, :, ::3] = -0.0
    k[5] = -0.0
    k[6] = 0.0
    c = KV4Cache(1, 1, D, device=DEV)
    c.append(k.to(DEV), k.to(DEV), torch.arange(64, device=DEV))
    codes, s8 = kv4.quantise(k[:, 0])
    assert torch.equal(c.pages[0, 0].cpu(), kv4.pack_page(codes, s8, codes, s8))


# ----------------------------------------------------------------------- tables wider than the sequences
@pytest.mark.parametrize("lens,news,H,G,D,dtype,window", [
    ([1000], [40], 1, 2, 128, torch.float16, 0),
    ([300, 1500], [33, 60], 2, 2, 64, torch.bfloat16, 0),
    ([2000, 100], [70, 100], 1, 2, 256, torch.float16, 0),
    ([1800], [50], 1, 4, 128, torch.bfloat16, 700),
    ([3, 1100], [40, 40], 1, 1, 128, torch.float16, 1090),
])
def test_a_table_padded_to_the_longest_length(KV4Cache, lens, news, H, G, D, dtype, window):
    """As a server has it.  A tile's keys are split by what it has, not by what the table could hold: the same bits
    whether the table is as wide as two or as sixty-four stretches, and whole."""
    got = []
    for width in (2048, 512):
        x = Batch(lens, news, H, G, D, dtype, seed=52, width=width)
        c = x.cache(KV4Cache)
        out, lse = c.attend(*x.args(), 0.1, max_q=64 // G + max(news), window=window, return_lse=True)
        c.check()
        check(out, lse, x.oracle(0.1, window), max(lens))
        got.append((out, lse))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


# ------------------------------------------------------------------------------- rows in one call or in several
@pytest.mark.parametrize("T", [1023, 1024, 4096, 4097])
@pytest.mark.parametrize("order", ["runs", "scattered", "mixed"])
def test_one_append_is_what_several_are(KV4Cache, T, order):
    """The bounds are looked for in other ways for few rows than for many: bytes, bounds and units are the same."""
    g = torch.Generator().manual_seed(T)
    P, H, D = 160, 2, 64
    perm = torch.randperm(P, generator=g)
    j = torch.arange(T)
    runs = perm[j // 64] * 64 + j % 64
    slots = {"runs": runs, "scattered": torch.randperm(P * 64, generator=g)[:T],
             "mixed": torch.cat([runs[:T // 2], (perm[T // 128 + 1:, None] * 64 + torch.randperm(64, generator=g)).flatten()[:T - T // 2]])}[order]
    assert len(slots.unique()) == T
    k, v = ((torch.randn(T, H, D, generator=g) * 2).bfloat16().to(DEV) for _ in range(2))
    slots = slots.to(DEV)
    one, many = KV4Cache(P, H, D, device=DEV), KV4Cache(P, H, D, device=DEV)
    one.append(k, v, slots)
    for i in range(0, T, 300):
        many.append(k[i:i + 300], v[i:i + 300], slots[i:i + 300])
    assert torch.equal(one.pages, many.pages) and torch.equal(one.bounds, many.bounds) and torch.equal(one.unit, many.unit)
    page = int(slots[T // 3]) // 64
    want, unit = kv4.bounds(one.read(torch.arange(page * 64, page * 64 + 64, device=DEV), torch.float16)[0][:, 1].float().cpu())
    assert torch.equal(one.bounds[page, 1].cpu(), want) and float(one.unit[page, 1]) == unit


@pytest.mark.parametrize("max_q", [2, 100])
@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16), (256, torch.float16)])
def test_unwritten_bytes_against_64_bits(KV4Cache, D, dtype, max_q):
    """Pages of 0xFF (NaN scales) but for the sequences' own rows: outputs within the bound of every other case."""
    x = Batch([70, 1, 190], [2, 1, 2], 1, 4, D, dtype, seed=53)
    c = KV4Cache(x.n_pages, 1, D, device=DEV)
    c.pages.fill_(0xFF)
    c.append(x.k.to(DEV), x.v.to(DEV), x.slots.to(DEV))
    out, lse = c.attend(*x.args(), 0.1, max_q=max_q, return_lse=True)
    check(out, lse, x.oracle(0.1), 190)
    pages = torch.tensor([[[1, 0]], [[0, 1]], [[0, -1]], [[2, 0]], [[1, 2]]], dtype=torch.int32)
    out, lse = c.attend(*x.args(), 0.1, max_q=max_q, pages=pages.to(DEV), return_lse=True)
    check(out, lse, x.oracle(0.1, pages=pages), 128)
    c.check()


def test_more_heads_than_a_grid_has_rows_are_refused(KV4Cache):
    """Before anything is written: the bounds could not be recomputed."""
    c = KV4Cache(1, 1, 64, device=DEV)
    c.pages = torch.zeros(1, 65536, 72 * 64, dtype=torch.uint8, device=DEV)
    c.bounds = torch.zeros(1, 65536, 2, 64, dtype=torch.int8, device=DEV)
    c.unit = torch.ones(1, 65536, device=DEV)
    k = torch.ones(1, 65536, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="65535"):
        c.append(k, k, torch.zeros(1, dtype=torch.int64, device=DEV))
    assert not c.pages.any()
