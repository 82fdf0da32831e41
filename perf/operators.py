"""Measured cases of the 4-bit paged K/V cache for grouped-query attention.

Five operators over one cache (`vllm_moet_b200.ops.kv4.KV4Cache`): rows are quantised as
they are written ("store", which also keeps the page bounds), read back ("load"), the pages
a query needs are chosen by a cheap score ("select"), and queries attend to every page of
their sequence ("attend") or to the chosen ones ("sparse" = select, then attend).

Each case runs either through the framework (`own` true) or in plain torch operations in 32
bits over an unpermuted copy of the same cache.

Formulas, for one row x of D values of one K/V head, in blocks of 16:
    s = e4m3(amax(|x_block|) / 6 * 64) / 64      (round to nearest even, at most 448 / 64)
    x^ = s * nearest of {0, .5, 1, 1.5, 2, 3, 4, 6} to |x| / s, ties to the even code, signed
For a page (64 positions) with key rows k^: hi_d = ceil(max k^_d / e), lo_d = floor(min k^_d / e),
e the smallest power of two, 2^-100 at least, with max |k^| <= 127 e (1 for a page of zeros).
Score of a page for a query token and a K/V head: the largest over the head's query rows of
    f * e * sum_d (max(r_d, 0) hi_d + min(r_d, 0) lo_d),  r = round(q / f), f as e for |q|.
Integers below 2^24 times powers of two: the score is exact, so the choice is one and the same.
Attention: softmax(scale * q . k^) v^ over positions j <= p, j > p - window, query i of n at
p = length - n + i; with chosen pages, over their positions only.  A row without positions
gives zeros and a log-sum-exp of -inf.
"""
import math
import random

import torch

own = False

PAGE = 64
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------- cases
def _case(name, op, **kw):
    base = dict(name=name, op=op, dtype="bf16", seqs=1, new=1, ctx=1024, ragged=False, kv_heads=8, group=8, dim=128,
                budget=0, window=0, mix=1)
    base.update(kw)
    return base


def listed():
    return [
        # one new token of each of 32 running sequences: the write of a decode step
        _case("store_step", "store", seqs=32, new=1, ctx=700, ragged=True, mix=3),
        # an 8192-token batch of prompts of uneven lengths, as prefill writes it
        _case("store_prompts", "store", seqs=6, new=4000, ctx=4000, ragged=True, mix=190),
        # a whole 32k context read back to 16 bits, for a prefill that continues it
        _case("load_context", "load", seqs=1, ctx=32768),
        # short uneven prefixes of a small-headed draft layer
        _case("load_prefixes", "load", dtype="f16", seqs=9, ctx=333, ragged=True, kv_heads=3, group=2, dim=64, mix=5),
        # decode: 32 sequences of up to 64k positions choose 64 pages for their next token
        _case("select_step", "select", seqs=32, ctx=65536, ragged=True, budget=64, mix=2),
        # a 1024-token chunk at the end of a 32k prompt chooses pages for every token
        _case("select_chunk", "select", seqs=1, new=1024, ctx=32768, budget=32),
        # one stream, a short context: latency
        _case("attend_one", "attend", seqs=1, ctx=1000, group=4),
        # 32 streams over long contexts of uneven lengths: the cache's bytes
        _case("attend_batch", "attend", seqs=32, ctx=32768, ragged=True, mix=7),
        # three verify rows of speculative decoding, wide heads, a sliding window, odd lengths and one
        # sequence shorter than its rows
        _case("attend_verify", "attend", dtype="f16", seqs=13, new=3, ctx=5001, ragged=True, kv_heads=2, group=5, dim=256,
              window=4000, mix=4),
        # a 2048-token chunk of a long prompt: matrix products
        _case("attend_chunk", "attend", seqs=1, new=2048, ctx=16384, group=4),
        # decode at 128k positions over 64 chosen pages
        _case("sparse_step", "sparse", seqs=8, ctx=131072, ragged=True, budget=64, mix=6),
        # a 333-token chunk with pages of its own for every token
        _case("sparse_chunk", "sparse", seqs=1, new=333, ctx=20011, budget=32, group=16, kv_heads=4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["store", "load", "select", "attend", "attend", "sparse"])
    case = dict(op=op, dtype=rng.choice(["bf16", "f16"]), kv_heads=rng.choice([1, 2, 3, 4, 8]),
                group=rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]), dim=rng.choice([64, 128, 128, 256]), ragged=rng.random() < 0.7,
                budget=0, window=0, mix=rng.randrange(1 << 20))
    case["seqs"] = _log(rng, 1, 48)
    prompt = rng.random() < 0.4
    case["new"] = _log(rng, 9, 2048) if prompt else rng.choice([1, 1, 2, 3, 5])
    row = case["kv_heads"] * case["dim"]
    case["ctx"] = _log(rng, 1, min(131072, (1 << 30) // (row * case["seqs"])))
    if op in ("select", "sparse"):
        case["budget"] = _log(rng, 3, 96)
    if op == "select":                                       # a choice to make: more pages than the budget
        case["seqs"] = min(case["seqs"], (1 << 30) // (row * PAGE * 2 * case["budget"]))
        case["ctx"] = max(case["ctx"], PAGE * 2 * case["budget"])
    if op == "attend" and rng.random() < 0.3:
        case["window"] = _log(rng, 1, case["ctx"])
    if op == "load":
        case["ctx"] = min(case["ctx"], max(1, (1 << 25) // (row * case["seqs"])))
    if op in ("select", "attend", "sparse"):
        case["new"] = min(case["new"], case["ctx"])
    # no more query rows than the largest listed case has score entries and gathered values for
    rows = case["seqs"] * case["kv_heads"] * case["group"]
    if op == "attend":
        case["new"] = max(1, min(case["new"], (1 << 30) // (rows * case["ctx"])))
    if op == "select":
        case["new"] = max(1, min(case["new"], (1 << 28) // (rows * (case["ctx"] // PAGE + 1))))
    if op == "sparse":
        gathered = case["seqs"] * row * PAGE * case["budget"]
        case["new"] = max(1, min(case["new"], (1 << 30) // gathered, (1 << 28) // (rows * (case["ctx"] // PAGE + 1))))
    if op == "store":
        case["new"] = max(1, min(case["new"], case["ctx"], (1 << 24) // (row * case["seqs"])))
    return case


def _lengths(case):
    """(positions, new rows) of each sequence: the case's own, the same for every seed."""
    rng = random.Random(case["mix"])
    lens, news = [], []
    for b in range(case["seqs"]):
        n, m = case["ctx"], case["new"]
        if case["ragged"] and b:
            n = _log(rng, max(1, case["ctx"] // 8), case["ctx"])
            m = rng.randint(max(1, case["new"] // 2), case["new"])
            if case["op"] == "attend" and b == 1:
                n = min(n, 2)                       # fewer positions than rows: empty rows
            elif case["op"] != "store":
                m = min(m, n)
        if case["op"] in ("store", "load"):
            m = min(m, n)
        lens.append(n)
        news.append(m)
    return lens, news


# -------------------------------------------------------------------------- the inputs
def _inputs(case, seed):
    """Raw keys / values of every position, the new rows (as slices of one projection's output,
    as a layer has them), page tables and lengths."""
    dev = "cuda"
    dt, H, G, D = TYPES[case["dtype"]], case["kv_heads"], case["group"], case["dim"]
    g = torch.Generator(device=dev).manual_seed(seed)
    lens, news = _lengths(case)
    widths = [-(-n // PAGE) for n in lens]
    pages = sum(widths) + 3
    perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(lens), max(widths), dtype=torch.int32, device=dev)
    slots, at, total = [], 0, 0
    for b, (n, w) in enumerate(zip(lens, widths)):
        table[b, :w] = perm[at:at + w]
        j = torch.arange(n, device=dev)
        slots.append(table[b, j // PAGE].long() * PAGE + j % PAGE)
        at, total = at + w, total + n
    # keys have channels of uneven size and a mean, as projections' outputs have; values do not
    gain = torch.exp(0.5 * torch.randn(H, D, generator=g, device=dev))
    mean = 0.5 * torch.randn(H, D, generator=g, device=dev)
    k = torch.randn(total, H, D, generator=g, device=dev, dtype=dt)
    k.mul_(gain.to(dt)).add_(mean.to(dt))
    v = torch.randn(total, H, D, generator=g, device=dev, dtype=dt)
    # the last positions' rows are the new ones
    where, at = [], 0
    for n, m in zip(lens, news):
        where.append(torch.arange(n - m, n, device=dev).clamp_(min=0) + at)
        at += n
    where = torch.cat(where)
    T = where.numel()
    qkv = torch.empty(T, H * (G + 2), D, device=dev, dtype=dt)
    qkv[:, :H * G] = 1.5 * torch.randn(T, H * G, D, generator=g, device=dev, dtype=dt)
    qkv[:, H * G:H * (G + 1)] = k[where]
    qkv[:, H * (G + 1):] = v[where]
    cu = [0]
    for m in news:
        cu.append(cu[-1] + m)
    return dict(k=k, v=v, slots=torch.cat(slots), new_slots=torch.cat(slots)[where], qkv=qkv, pages=pages,
                q=qkv[:, :H * G], k_new=qkv[:, H * G:H * (G + 1)], v_new=qkv[:, H * (G + 1):],
                cu_q=torch.tensor(cu, dtype=torch.int32, device=dev),
                seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev), table=table, max_q=max(news),
                scale=D ** -0.5)


def prepare(case, seed):
    x = _inputs(case, seed)
    k, v = x.pop("k"), x.pop("v")
    if own:
        from vllm_moet_b200.ops.kv4 import KV4Cache
        cache = KV4Cache(x["pages"], case["kv_heads"], case["dim"], device="cuda")
        cache.append(k, v, x["slots"])
    else:
        cache = _plain_cache(x["pages"], case["kv_heads"], case["dim"])
        _plain_store(cache, k, v, x["slots"])
    if case["op"] == "load":
        x["new_slots"] = x["slots"]
    return dict(x, case=case, cache=cache)


# --------------------------------------------------------------------- the plain forms
def _plain_cache(pages, H, D):
    def z(*shape, dtype=torch.uint8):
        return torch.zeros(*shape, dtype=dtype, device="cuda")
    return dict(k=z(pages * PAGE, H, D // 2), ks=z(pages * PAGE, H, D // 16), v=z(pages * PAGE, H, D // 2),
                vs=z(pages * PAGE, H, D // 16), bounds=z(pages, H, 2, D, dtype=torch.int8),
                unit=torch.ones(pages, H, device="cuda"))


def _quantise(x):
    """[..., D] -> codes [..., D / 2] (even dim in the low half), scale bytes [..., D / 16]."""
    x = x.float().unflatten(-1, (-1, 16))
    s8 = (x.abs().amax(-1) / 6 * 64).clamp(max=448).to(torch.float8_e4m3fn)
    s = (s8.float() / 64)[..., None]
    a = x.abs()
    code = ((a > 0.25 * s).to(torch.uint8) + (a >= 0.75 * s) + (a > 1.25 * s) + (a >= 1.75 * s) + (a > 2.5 * s)
            + (a >= 3.5 * s) + (a > 5 * s))
    code = (torch.where(s > 0, code, 0) | ((x < 0).to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), s8.view(torch.uint8)


def _values(codes, scales):
    e2m1 = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    pair = torch.stack([e2m1.repeat(16), e2m1.repeat_interleave(16)], -1)
    x = pair[codes.int()].flatten(-2).unflatten(-1, (-1, 16))
    return (x * (scales.view(torch.float8_e4m3fn).float() / 64)[..., None]).flatten(-2)


def _power(amax):
    """The smallest power of two e >= 2^-100 with amax <= 127 e, 1 for amax = 0."""
    m, x = torch.frexp(amax)
    x = (x - 7 + (m > 127 / 128).int()).clamp(min=-100)
    return torch.where(amax > 0, ((x + 127) << 23).view(torch.float32), 1.0)


def _plain_store(c, k, v, slots):
    c["k"][slots], c["ks"][slots] = _quantise(k)
    c["v"][slots], c["vs"][slots] = _quantise(v)
    page = slots // PAGE
    page = page[torch.cat([page[1:] != page[:-1], torch.ones_like(page[:1], dtype=torch.bool)])]
    rows = page[:, None] * PAGE + torch.arange(PAGE, device=page.device)
    x = _values(c["k"][rows], c["ks"][rows])
    hi, lo = x.amax(1), x.amin(1)
    e = _power(torch.maximum(hi.abs(), lo.abs()).amax(-1))
    c["bounds"][page] = torch.stack([torch.ceil(hi / e[..., None]), torch.floor(lo / e[..., None])], 2).to(torch.int8)
    c["unit"][page] = e


def _rows(s):
    """(sequence, index in it, position) of each query row."""
    t = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.bucketize(t, s["cu_q"][1:], right=True)
    i = t - s["cu_q"][b]
    return b, i, s["seq_lens"][b] - (s["cu_q"][b + 1] - s["cu_q"][b]) + i


def _padded(s, x):
    """x [T, ...] by sequence: [B, max_q, ...]; rows past a sequence's own repeat others."""
    at = s["cu_q"][:-1, None] + torch.arange(s["max_q"], device="cuda")
    return x[at.clamp(max=x.shape[0] - 1)]


def _plain_select(s):
    """The budget's pages of each token and head, ascending, -1 where there are fewer."""
    c, case = s["cache"], s["case"]
    H, G = case["kv_heads"], case["group"]
    q = s["q"].float().unflatten(1, (H, G))
    f = _power(q.abs().amax(-1))[..., None]
    r = torch.round(q / f)
    r = _padded(s, torch.cat([r.clamp(min=0), r.clamp(max=0)], -1))           # [B, n, H, G, 2D]
    table = s["table"].long()
    bound = c["bounds"][table].float().flatten(-2)                            # [B, W, H, 2D]
    score = torch.matmul(r.permute(0, 2, 1, 3, 4).flatten(2, 3), bound.permute(0, 2, 3, 1)).unflatten(2, (-1, G))
    score = score * _padded(s, f).permute(0, 2, 1, 3, 4) * c["unit"][table].transpose(1, 2)[:, :, None, None]
    b, i, pos = _rows(s)
    score = score.amax(3).transpose(1, 2)[b, i]                               # [T, H, W]
    last = (pos // PAGE)[:, None, None]
    w = torch.arange(score.shape[-1], device="cuda")
    score = torch.where((w < 1) | (w >= last - 1), math.inf, score)           # the first and the last two pages
    score = torch.where((w > last) | (pos < 0)[:, None, None], -math.inf, score)
    best = torch.sort(score, dim=-1, descending=True, stable=True)
    n = min(case["budget"], score.shape[-1])
    idx = torch.where(best.values[..., :n] == -math.inf, score.shape[-1], best.indices[..., :n]).sort(-1).values
    idx = torch.where(idx == score.shape[-1], -1, idx).int()
    return torch.nn.functional.pad(idx, (0, case["budget"] - n), value=-1)


def _softmax_av(score, seen, v):
    """softmax of score over the last axis where `seen`, times v, and its log-sum-exp."""
    score = score.masked_fill(~seen, -math.inf)
    m = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - m)
    z = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / z.clamp(min=1e-30), (m + torch.log(z)).squeeze(-1)


def _plain_attend(s):
    c, case = s["cache"], s["case"]
    H, G = case["kv_heads"], case["group"]
    q = _padded(s, s["q"].float().unflatten(1, (H, G))).permute(0, 2, 1, 3, 4)    # [B, H, n, G, D]
    rows = (s["table"].long()[..., None] * PAGE + torch.arange(PAGE, device="cuda")).flatten(1)
    k = _values(c["k"][rows], c["ks"][rows]).permute(0, 2, 3, 1)                  # [B, H, D, L]
    v = _values(c["v"][rows], c["vs"][rows]).transpose(1, 2)
    score = torch.matmul(q.flatten(2, 3), k) * s["scale"]
    j = torch.arange(rows.shape[1], device="cuda")
    b, i, pos = _rows(s)
    n = s["cu_q"][1:] - s["cu_q"][:-1]
    p = (s["seq_lens"] - n)[:, None] + torch.arange(s["max_q"], device="cuda")
    seen = j <= p[..., None]
    if case["window"]:
        seen &= j > p[..., None] - case["window"]
    out, lse = _softmax_av(score, seen.repeat_interleave(G, 1)[:, None], v)
    out, lse = out.unflatten(2, (-1, G))[b, :, i], lse.unflatten(2, (-1, G))[b, :, i]
    return out.flatten(1, 2).to(s["q"].dtype), lse.flatten(1, 2)


def _plain_sparse(s, pages):
    c, case = s["cache"], s["case"]
    H, G = case["kv_heads"], case["group"]
    b, _, pos = _rows(s)
    j = (pages[..., None] * PAGE + torch.arange(PAGE, device="cuda")).flatten(2)      # positions [T, H, L]
    phys = s["table"][b[:, None, None], pages.clamp(min=0).long()].long()
    rows = (phys[..., None] * PAGE + torch.arange(PAGE, device="cuda")).flatten(2)
    h = torch.arange(H, device="cuda")[:, None]
    k = _values(c["k"][rows, h], c["ks"][rows, h])
    v = _values(c["v"][rows, h], c["vs"][rows, h])                                    # [T, H, L, D]
    q = s["q"].float().unflatten(1, (H, G))
    seen = (j >= 0) & (j <= pos[:, None, None]) & (pages >= 0).repeat_interleave(PAGE, 2)
    out, lse = _softmax_av(torch.matmul(q, k.transpose(2, 3)) * s["scale"], seen[:, :, None], v)
    return out.flatten(1, 2).to(s["q"].dtype), lse.flatten(1, 2)


# --------------------------------------------------------------------------- one pass
def _run_own(s):
    c, case, op = s["cache"], s["case"], s["case"]["op"]
    batch = (s["q"], s["cu_q"], s["seq_lens"], s["table"])
    if op == "store":
        c.append(s["k_new"], s["v_new"], s["new_slots"])
        k, v = c.read(s["new_slots"], s["q"].dtype)
        return dict(k=k, v=v, bounds=c.bounds, unit=c.unit)
    if op == "load":
        k, v = c.read(s["new_slots"], s["q"].dtype)
        return dict(k=k, v=v)
    pages = None
    if op in ("select", "sparse"):
        pages = c.select(*batch, case["budget"], max_q=s["max_q"])
        if op == "select":
            return dict(pages=pages)
    out, lse = c.attend(*batch, s["scale"], max_q=s["max_q"], window=case["window"], pages=pages, return_lse=True)
    return dict(out=out, lse=lse) if pages is None else dict(out=out, lse=lse, pages=pages)


def run(state):
    if own:
        return _run_own(state)
    s, c, op = state, state["cache"], state["case"]["op"]
    if op == "store":
        _plain_store(c, s["k_new"], s["v_new"], s["new_slots"])
    if op in ("store", "load"):
        dt, at = s["q"].dtype, s["new_slots"]
        got = dict(k=_values(c["k"][at], c["ks"][at]).to(dt), v=_values(c["v"][at], c["vs"][at]).to(dt))
        return dict(got, bounds=c["bounds"], unit=c["unit"]) if op == "store" else got
    if op == "attend":
        out, lse = _plain_attend(s)
        return dict(out=out, lse=lse)
    pages = _plain_select(s)
    if op == "select":
        return dict(pages=pages)
    out, lse = _plain_sparse(s, pages)
    return dict(out=out, lse=lse, pages=pages)


# ---------------------------------------------------------------- what a pass has to do
def work(case):
    lens, news = _lengths(case)
    H, G, D = case["kv_heads"], case["group"], case["dim"]
    row4 = H * D * 9 // 16                                   # a position's keys (or values) in the cache
    T, op = sum(news), case["op"]
    if op == "store":
        touched = sum(-(-m // PAGE) for m in news) * H * (2 * D + 4)
        return dict(bytes=T * (4 * H * D + 2 * row4 + 8) + touched + T * (2 * row4 + 4 * H * D + 8), flops=T * H * D * 8)
    if op == "load":
        return dict(bytes=sum(lens) * (2 * row4 + 4 * H * D + 8), flops=2 * sum(lens) * H * D)
    q = 2 * T * H * G * D
    nbytes, flops = q, 0
    if op in ("select", "sparse"):
        n = sum(-(-x // PAGE) for x in lens)
        nbytes += n * H * (2 * D + 4) + 4 * T * H * case["budget"]
        flops += sum(2 * 2 * D * H * G * m * (x // PAGE) for x, m in zip(lens, news))
    if op in ("attend", "sparse"):
        nbytes += q + 4 * T * H * G                           # outputs and their log-sum-exps
    if op == "attend":
        w = case["window"] or case["ctx"]
        nbytes += sum(min(x, w + m - 1) for x, m in zip(lens, news)) * 2 * row4
        pairs = sum(max(0, min(w, x - m + i + 1)) for x, m in zip(lens, news) for i in range(m))
        flops += 4 * D * H * G * pairs
    if op == "sparse":
        cap = PAGE * case["budget"]
        nbytes += sum(min(x, m * cap) for x, m in zip(lens, news)) * 2 * row4
        flops += 4 * D * H * G * sum(m * min(x, cap) for x, m in zip(lens, news))
    return dict(bytes=nbytes, flops=flops)


# ---------------------------------------------------- the definition, in 64 bits, apart
def _nearest(x):
    """The value that a block-16 row's element is held as, by search over every code."""
    y = x.double().reshape(-1, 16)
    top = y.abs().max(1).values
    grid = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    want = (top * 64 / 6).clamp(max=448.0)
    hi = torch.searchsorted(grid, want).clamp(1, 126)
    up, down = grid[hi] - want, want - grid[hi - 1]
    s = grid[torch.where((down < up) | ((down == up) & (hi % 2 == 1)), hi - 1, hi)] / 64
    mags = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    held = torch.zeros_like(y)
    gap = torch.full_like(y, math.inf)
    for code in (0, 2, 4, 6, 1, 3, 5, 7):                    # even codes first: they keep their ties
        d = (y.abs() - mags[code] * s[:, None]).abs()
        held = torch.where(d < gap, mags[code] * s[:, None], held)
        gap = torch.minimum(gap, d)
    return (torch.sign(y) * held).reshape(x.shape)


def _two(amax):
    def power(e):                                            # by its bits: a library's pow may be off by one
        return ((e.long() + 1023) << 52).view(torch.float64)
    e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -93) / 127)).clamp(min=-100)
    e = torch.where((127 * power(e - 1) >= amax) & (e > -100), e - 1, e)
    e = torch.where(127 * power(e) < amax, e + 1, e)
    return torch.where(amax > 0, power(e), torch.ones_like(amax))


def exact(case, seed):
    lens, news = _lengths(case)
    H, G, D, op = case["kv_heads"], case["group"], case["dim"], case["op"]
    x = _inputs(case, seed)
    starts = [sum(lens[:b]) for b in range(len(lens))]
    if op == "load":
        return dict(k=_nearest(x["k"]), v=_nearest(x["v"]))
    if op == "store":
        bounds = torch.zeros(x["pages"], H, 2, D, dtype=torch.int8, device="cuda")
        unit = torch.ones(x["pages"], H, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            w = -(-n // PAGE)
            held = torch.zeros(w * PAGE, H, D, dtype=torch.float64, device="cuda")   # not written yet: zeros
            held[:n] = _nearest(x["k"][starts[b]:starts[b] + n])
            held = held.reshape(w, PAGE, H, D)
            e = _two(held.abs().amax(1).amax(-1))
            page = x["table"][b, :w].long()
            bounds[page, :, 0] = torch.ceil(held.amax(1) / e[..., None]).to(torch.int8)
            bounds[page, :, 1] = torch.floor(held.amin(1) / e[..., None]).to(torch.int8)
            unit[page] = e
        return dict(k=_nearest(x["k_new"]), v=_nearest(x["v_new"]), bounds=bounds, unit=unit)
    outs, lses, chosen = [], [], []
    at = 0
    for b, (n, m) in enumerate(zip(lens, news)):
        q = x["q"][at:at + m].double().reshape(m, H, G, D)
        at += m
        w = -(-n // PAGE)
        pos = torch.arange(n - m, n, device="cuda")
        k = torch.cat([_nearest(x["k"][starts[b]:starts[b] + n]),
                       torch.zeros(w * PAGE - n, H, D, dtype=torch.float64, device="cuda")])
        keep = None
        if op in ("select", "sparse"):
            kp = k.reshape(w, PAGE, H, D)
            e = _two(kp.abs().amax(1).amax(-1))[..., None]
            hi, lo = torch.ceil(kp.amax(1) / e) * e, torch.floor(kp.amin(1) / e) * e
            f = _two(q.abs().amax(-1))[..., None]
            r = torch.round(q / f) * f
            score = (torch.einsum("mhgd,whd->mhgw", r.clamp(min=0), hi)
                     + torch.einsum("mhgd,whd->mhgw", r.clamp(max=0), lo)).amax(2)
            page = torch.arange(w, device="cuda")
            last = (torch.div(pos, PAGE, rounding_mode="floor"))[:, None, None]
            score[((page == 0) | (page == last) | (page == last - 1)).expand_as(score)] = math.inf
            score[(page > last).expand_as(score)] = -math.inf
            order = torch.argsort(score, dim=-1, descending=True, stable=True)[..., :case["budget"]]
            keep = torch.zeros_like(score, dtype=torch.bool).scatter_(2, order, True) & (score > -math.inf)
            names = torch.where(keep, page, w).sort(-1).values[..., :case["budget"]]
            names = torch.where(names == w, -1, names).int()
            chosen.append(torch.nn.functional.pad(names, (0, case["budget"] - names.shape[-1]), value=-1))
            if op == "select":
                continue
        v = _nearest(x["v"][starts[b]:starts[b] + n])
        for h in range(H):
            score = torch.einsum("mgd,nd->mgn", q[:, h], k[:n, h]) * x["scale"]
            j = torch.arange(n, device="cuda")
            hide = j > pos[:, None]
            if case["window"]:
                hide |= j <= pos[:, None] - case["window"]
            if keep is not None:
                hide |= ~keep[:, h].repeat_interleave(PAGE, -1)[:, :n]
            score = score.masked_fill(hide[:, None], -math.inf)
            lse = torch.logsumexp(score, -1)
            p = torch.exp(score - torch.where(lse == -math.inf, 0.0, lse)[..., None])
            outs.append((b, torch.einsum("mgn,nd->mgd", p, v[:, h])))
            lses.append(lse)
    got = {}
    if chosen:
        got["pages"] = torch.cat(chosen)
    if outs:
        def by_row(parts):
            return torch.cat([torch.cat(parts[b * H:(b + 1) * H], 1) for b in range(len(lens))])
        got["out"], got["lse"] = by_row([o for _, o in outs]), by_row(lses)
    return got
