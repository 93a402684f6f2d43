"""The 8-bit paged cache and attention over it against their definitions in 64 bits (tests/_cache_util.py)."""
import math

import pytest
import torch

import flashmask_b200 as fm
import _cache_util as ref

pytestmark = pytest.mark.gpu
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def values_of(payload):
    return payload.cpu().float().double()


class Filled:
    """A cache with B sequences of the given lengths, random pages, and the same contents in 64 bits."""

    def __init__(self, lens, H, d, dv, kind=E4M3, page=16, seed=0, spare=2, dtype=torch.bfloat16, table_pages=None):
        g = torch.Generator().manual_seed(seed)
        need = [-(-max(n, 1) // page) for n in lens]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g)
        width = table_pages or max(need)
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.lens, self.page, self.kind = lens, page, kind
        self.cache = fm.QuantizedKVCache.empty(pages, H, d, dv, page_size=page, dtype=kind)
        # every page gets its own magnitude, so that scales differ
        for name, w in (("k", d), ("v", dv)):
            x = torch.randn(pages, H, page, w, generator=g) * torch.exp(0.7 * torch.randn(pages, H, 1, 1, generator=g))
            scale = torch.tensor([[2.0 ** ref.least_exponent(float(x[p, h].to(dtype).abs().max()), kind) for h in range(H)] for p in range(pages)])
            q = ref.grid(x.to(dtype).double() / scale.double()[..., None, None], kind)
            getattr(self.cache, name).copy_((q.float().to(kind) if kind == E4M3 else q.to(kind)).cuda())
            getattr(self.cache, name + "_scale").copy_(scale.cuda())
        self.seqlens = torch.tensor(lens, dtype=torch.int32)

    def largest_scale(self, b):
        own = [p for p in self.table[b].tolist() if 0 <= p < self.cache.k.shape[0]]
        s = self.cache.v_scale.cpu()[own]
        return float(s[torch.isfinite(s)].max()) if len(own) else 0.0

    def dense(self, b, name, n=None):
        return ref.dense(values_of(getattr(self.cache, name)), getattr(self.cache, name + "_scale").cpu().double(), self.table[b],
                         self.lens[b] if n is None else n)


def check_attention(f, q, *, q_lengths=None, causal=True, window=None, scale=None, sink=None, got=None, **kw):
    B, S, Hq, d = q.shape
    if got is None:
        got = fm.kv_cache_attention(q.cuda(), f.cache, f.table.cuda(), f.seqlens.cuda(), causal=causal, window_size=window,
                                    q_lengths=None if q_lengths is None else torch.tensor(q_lengths, dtype=torch.int32).cuda(),
                                    softmax_scale=scale, sink=None if sink is None else sink.cuda(), return_lse=True, **kw)
    out, lse = got[0].cpu().double(), got[1].cpu().double()
    half = torch.finfo(q.dtype).eps / 2
    for b in range(B):
        cap = f.table.shape[1] * f.page
        n = min(max(f.lens[b], 0), cap)
        (k, there), (v, _) = f.dense(b, "k", n), f.dense(b, "v", n)
        rows = S if q_lengths is None else min(max(q_lengths[b], 0), S)
        o, l, weight, reach = ref.attention(q[b].double(), k, v, there, rows, causal, window, 1 / math.sqrt(d) if scale is None else scale, sink)
        # p is rounded to 16 bits (half a step is 2^-8 where the dense forward in bf16 takes the call, else 2^-11 in fp16); a
        # score is off by d steps of 2^-23 of the sum of its products' magnitudes (q in fp16: 2^-24 of its row's largest), a sum over
        # n keys by n steps of 2^-24
        p_half = 2.0 ** -8 if S * Hq // f.cache.k.shape[1] > 96 and q.dtype == torch.bfloat16 else 2.0 ** -11
        slack = reach * (d + 16) * 2.0 ** -23 + 2.0 ** -20 + max(n, 1) * 2.0 ** -24
        # (below the smallest normal number of the type half a step is no longer relative: smallest normal * eps / 2, 2^-25 in fp16)
        # (fp16's half step is 2^-25 for p below 2^-14, when the largest p is 2^7 at least: 2^-32 of the largest p_j vs_j for every
        # payload value, at most 448; the dense forward in bf16 has the same relative step everywhere, in fp16 2^-25 of the largest p)
        tol = half * o.abs() + n * 2.0 ** (-32 if S * Hq // f.cache.k.shape[1] <= 96 else -25) * 448 * f.largest_scale(b) + weight * (p_half + 2 * slack[..., None]) + torch.finfo(q.dtype).smallest_normal * half
        far = (out[b] - o).abs() - tol
        w = far.argmax()
        assert far.flatten()[w] <= 0, (b, int(w), *(t.flatten()[w].item() for t in (far, out[b], o, weight)))
        fin = torch.isfinite(l)
        assert torch.equal(torch.isinf(lse[b]), ~fin), b
        ltol = (slack.T + 2.0 ** -21 * l.abs())[fin] + 2.0 ** -20
        assert ((lse[b] - l).abs()[fin] <= ltol).all(), (b, (lse[b] - l).abs()[fin].max())
    return got


def rand_q(B, S, Hq, d, seed=1, dtype=torch.bfloat16, size=1.0):
    return (size * torch.randn(B, S, Hq, d, generator=torch.Generator().manual_seed(seed))).to(dtype)


# ------------------------------------------------------------------ writing and reading
@pytest.mark.parametrize("kind", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,d,dv,H", [(16, 16, 16, 1), (16, 80, 48, 3), (32, 64, 128, 2), (64, 128, 128, 2), (128, 192, 128, 1), (128, 256, 256, 1)])
def test_write_is_exact_and_reads_back(kind, dtype, page, d, dv, H):
    f = Filled([3 * page + 5, 1, 2 * page], H, d, dv, kind, page, seed=2, dtype=dtype, table_pages=5)
    g = torch.Generator().manual_seed(3)
    S = page + 7
    # whole pages, a start inside a page, rows that do not count, a start before 0
    start, lengths = [page - 3, 0, page // 2], [S, 1, S - 6]
    for values, table in ((1.0, f.table), (300.0, f.table)):
        k = (values * torch.randn(3, S, H, d, generator=g)).to(dtype)
        v = (values * torch.randn(3, S, H, dv, generator=g) * torch.tensor([1.0, 1e-3, 30.0])[:, None, None, None]).to(dtype)
        want = {}
        for name, x in (("k", k), ("v", v)):
            vals, sc = values_of(getattr(f.cache, name)), getattr(f.cache, name + "_scale").cpu().double()
            ref.write((vals, kind), sc, x, table, start, lengths)
            want[name] = (vals, sc)
        fm.kv_cache_write(f.cache, k.cuda(), v.cuda(), table.cuda(), torch.tensor(start, dtype=torch.int32).cuda(),
                          torch.tensor(lengths, dtype=torch.int32).cuda())
        for name in ("k", "v"):
            assert torch.equal(getattr(f.cache, name + "_scale").cpu().double(), want[name][1]), name
            assert torch.equal(values_of(getattr(f.cache, name)), want[name][0]), name
    lens = [s + n for s, n in zip(start, lengths)]
    at = [5, -4, 0]
    got = fm.kv_cache_read(f.cache, f.table.cuda(), torch.tensor(at, dtype=torch.int32).cuda(),
                           torch.tensor(lens, dtype=torch.int32).cuda(), 2 * page + 3, dtype=dtype)
    for name, x in zip(("k", "v"), got):
        for b in range(3):
            dense, _ = f.dense(b, name, lens[b])
            full = torch.zeros(2 * page + 3, *dense.shape[1:], dtype=torch.float64)
            for i in range(2 * page + 3):
                if 0 <= at[b] + i < lens[b]:
                    full[i] = dense[at[b] + i]
            if dtype == torch.float16:
                full = full.clamp(-65504, 65504)
            assert torch.equal(x[b].cpu(), full.to(dtype)), (name, b)


@pytest.mark.parametrize("kind", [E4M3, INT8])
@pytest.mark.parametrize("page,d,dv,H", [(64, 32, 32, 3), (32, 64, 64, 5), (16, 192, 128, 3), (16, 256, 256, 3), (64, 64, 64, 1), (128, 128, 128, 1), (64, 256, 256, 1),
                                         (64, 112, 16, 2)])
def test_pages_that_warps_or_ctas_take(kind, page, d, dv, H):
    """Pages from a warp's share to a CTA's, heads that do not fill a CTA of warps, widths that leave lanes over."""
    test_write_is_exact_and_reads_back(kind, torch.bfloat16, page, d, dv, H)


@pytest.mark.parametrize("kind", [E4M3, INT8])
def test_tokens_appended_one_by_one(kind):
    """Scales that grow while a page fills, from tiny to large and back, and stay when they need not."""
    H, d, page = 2, 32, 16
    f = Filled([0, 0], H, d, d, kind, page, seed=4, table_pages=3)
    f.table[1] = -1
    f.table[0] = torch.tensor([1, 0, -1])
    g = torch.Generator().manual_seed(5)
    vals = {n: values_of(getattr(f.cache, n)) for n in "kv"}
    sc = {n: getattr(f.cache, n + "_scale").cpu().double() for n in "kv"}
    for step in range(2 * page):
        x = {n: (torch.randn(2, 1, H, d, generator=g) * 2.0 ** ((step * 7) % 23 - 11)).bfloat16() for n in "kv"}
        for n in "kv":
            ref.write((vals[n], kind), sc[n], x[n], f.table, [step, step], None)
        fm.kv_cache_write(f.cache, x["k"].cuda(), x["v"].cuda(), f.table.cuda(), torch.full((2,), step, dtype=torch.int32).cuda())
    for n in "kv":
        assert torch.equal(getattr(f.cache, n + "_scale").cpu().double(), sc[n])
        assert torch.equal(values_of(getattr(f.cache, n)), vals[n])


@pytest.mark.parametrize("kind", [E4M3, INT8])
def test_extreme_values(kind):
    """Zeros, subnormals, the ends of bf16's range, infinities and NaN."""
    d, page = 16, 16
    cache = fm.QuantizedKVCache.empty(4, 1, d, page_size=page, dtype=kind)
    tiny, huge = 2.0 ** -133, float(torch.finfo(torch.bfloat16).max)
    rows = [[0.0], [tiny, -tiny], [huge, -huge, 1.0], [1.0, math.inf, 2.0], [math.nan, 1.0]]
    x = torch.zeros(5, 1, 1, d)
    for i, r in enumerate(rows):
        x[i, 0, 0, :len(r)] = torch.tensor(r)
    x = x.bfloat16()
    for i in range(5):
        table = torch.tensor([[i % 4]], dtype=torch.int32)
        vals, sc = values_of(cache.k), cache.k_scale.cpu().double()
        ref.write((vals, kind), sc, x[i:i + 1], table, [0], None)
        fm.kv_cache_write(cache, x[i:i + 1].cuda(), x[i:i + 1].cuda(), table.cuda(), torch.zeros(1, dtype=torch.int32).cuda())
        assert torch.allclose(cache.k_scale.cpu().double(), sc, rtol=0, atol=0, equal_nan=True), i
        assert torch.allclose(values_of(cache.k), vals, rtol=0, atol=0, equal_nan=True), i
        back = fm.kv_cache_read(cache, table.cuda(), torch.zeros(1, dtype=torch.int32).cuda(), torch.ones(1, dtype=torch.int32).cuda(), 1)[0]
        bad = ~torch.isfinite(x[i]).flatten()
        assert torch.isnan(back.cpu().flatten()[bad]).all()
        if kind == E4M3 or not bad.any():
            assert torch.isfinite(back.cpu().flatten()[~bad]).all()
    # int8: the poisoned page stays NaN while it is appended to, and begins anew at slot 0
    one = torch.ones(1, 1, 1, d).bfloat16().cuda()
    t = torch.tensor([[0]], dtype=torch.int32).cuda()
    fm.kv_cache_write(cache, one, one, t, torch.ones(1, dtype=torch.int32).cuda())
    assert bool(torch.isnan(cache.k_scale[0, 0])) == (kind == INT8)
    fm.kv_cache_write(cache, one, one, t, torch.zeros(1, dtype=torch.int32).cuda())
    assert torch.isfinite(cache.k_scale[0, 0])


def test_write_leaves_the_rest_alone():
    """Pages of the table that the rows do not reach, pages of nobody, slots behind the last token, bad page numbers."""
    f = Filled([64, 64], 2, 64, 64, E4M3, 16, seed=6)
    n_pages = f.cache.k.shape[0]
    before = {n: getattr(f.cache, n).view(torch.uint8).clone() for n in "kv"}
    scales = {n: getattr(f.cache, n + "_scale").clone() for n in "kv"}
    table = f.table.clone()
    table[0, 2], table[1, 1], table[1, 2] = n_pages, -5, 2 ** 31 - 1
    x = torch.randn(2, 40, 2, 64).bfloat16().cuda()
    fm.kv_cache_write(f.cache, x, x, table.cuda(), torch.tensor([20, 10], dtype=torch.int32).cuda(), torch.tensor([13, 40], dtype=torch.int32).cuda())
    # sequence 0 wrote positions 20 .. 32: slots 4 .. 15 of page 1, and slot 0 of page 2, which is none;
    # sequence 1 positions 10 .. 49: slots 10 .. 15 of page 0, pages 1 and 2, which are none, slots 0, 1 of page 3
    touched = {int(f.table[0, 1]): (4, 16), int(f.table[1, 0]): (10, 16), int(f.table[1, 3]): (0, 2)}
    for n in "kv":
        now, same = getattr(f.cache, n).view(torch.uint8), torch.ones(n_pages, dtype=torch.bool)
        for p, (lo, hi) in touched.items():
            same[p] = False
            assert torch.equal(now[p, :, hi:], before[n][p, :, hi:])
            assert not torch.equal(now[p, :, lo:hi], before[n][p, :, lo:hi])
        assert torch.equal(now[same.cuda()], before[n][same.cuda()])
        assert torch.equal(getattr(f.cache, n + "_scale")[same.cuda()], scales[n][same.cuda()])


def test_write_takes_strided_views_and_starts_before_zero():
    f = Filled([40], 2, 64, 64, E4M3, 16, seed=7)
    g = Filled([40], 2, 64, 64, E4M3, 16, seed=7)
    wide = torch.randn(1, 24, 6, 64).bfloat16().cuda()
    k, v = wide[:, :, 1:3], wide[:, :, 4:6]
    start = torch.tensor([-5], dtype=torch.int32).cuda()
    fm.kv_cache_write(f.cache, k, v, f.table.cuda(), start)
    fm.kv_cache_write(g.cache, k[:, 5:].contiguous(), v[:, 5:].contiguous(), g.table.cuda(), start + 5)
    odd = torch.randn(1, 24, 2, 65).bfloat16().cuda()[..., 1:]            # rows that 16-byte vectors cannot read
    for n in "kv":
        assert torch.equal(getattr(f.cache, n).view(torch.uint8), getattr(g.cache, n).view(torch.uint8))
    fm.kv_cache_write(f.cache, odd, odd, f.table.cuda(), start + 5)
    fm.kv_cache_write(g.cache, odd.contiguous(), odd.contiguous(), g.table.cuda(), start + 5)
    for n in "kv":
        assert torch.equal(getattr(f.cache, n).view(torch.uint8), getattr(g.cache, n).view(torch.uint8))


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("kind", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,G,d,dv,page", [(1, 1, 16, 16, 16), (2, 4, 64, 64, 32), (2, 8, 80, 48, 16), (3, 5, 96, 128, 64), (2, 4, 128, 128, 64),
                                           (1, 16, 128, 64, 128), (2, 2, 192, 128, 64), (1, 9, 256, 256, 16)])
def test_one_token(kind, dtype, H, G, d, dv, page):
    f = Filled([1, 15, 16, 17, 130, 700, 0], H, d, dv, kind, page, seed=8, dtype=dtype)
    check_attention(f, rand_q(7, 1, H * G, d, dtype=dtype))


@pytest.mark.parametrize("S,G,causal,window", [(2, 4, True, None), (5, 4, True, 20), (3, 1, True, 1), (8, 8, True, 100), (7, 3, False, None),
                                               (16, 1, True, None), (33, 1, False, None), (64, 1, True, 33), (5, 4, False, None), (6, 4, True, 7), (24, 4, True, 50)])
def test_a_few_tokens(S, G, causal, window):
    """Fewer tokens than rows, rows that see nothing, windows inside and beyond the sequence."""
    f = Filled([max(S - 2, 1), S, S + 17, 333, 0, 1], 2, 128, 128, E4M3, 32, seed=9)
    check_attention(f, rand_q(6, S, 2 * G, 128), causal=causal, window=window)
    check_attention(f, rand_q(6, S, 2 * G, 128), causal=causal, window=window, sink=torch.randn(2 * G, generator=torch.Generator().manual_seed(4)))


@pytest.mark.parametrize("S", [4, 40])
@pytest.mark.parametrize("causal,window", [(True, None), (True, 9), (False, None)])
def test_padded_queries(S, causal, window):
    """Rows behind q_lengths are padding; 40 x 4 rows go through the dense forward, 4 x 4 do not."""
    lens = [50, 3, 200, 64, 0, 41]
    f = Filled(lens, 2, 64, 64, INT8, 16, seed=10, dtype=torch.float16)
    n = [1, 3, S, S - 1, 0, S + 5]
    for sink in (None, torch.linspace(-2, 3, 8)):
        out, lse = check_attention(f, rand_q(6, S, 8, 64, dtype=torch.float16), q_lengths=n, causal=causal, window=window, sink=sink)
        for b in range(6):
            assert not out[b, max(min(n[b], S), 0):].any()


@pytest.mark.parametrize("kind", [E4M3, INT8])
@pytest.mark.parametrize("d,dv,dtype", [(128, 128, torch.bfloat16), (64, 64, torch.float16), (192, 128, torch.bfloat16), (256, 256, torch.float16)])
def test_a_chunk_of_a_prompt(kind, d, dv, dtype):
    """More rows than the kernel for few takes: ragged lengths, a length below the chunk's, an upper bound or none."""
    f = Filled([150, 37, 300], 2, d, dv, kind, 64, seed=11, dtype=dtype)
    q = rand_q(3, 40, 8, d, dtype=dtype)
    a = check_attention(f, q)
    check_attention(f, q, window=30, sink=torch.randn(8, generator=torch.Generator().manual_seed(4)))
    b = check_attention(f, q, max_seqlen=300)
    assert torch.allclose(a[0].float(), b[0].float(), rtol=2e-2, atol=2e-2)


def test_many_rows_of_a_wide_table_take_no_dense_tensors():
    """Without an upper bound of the lengths and with a page table of 2 M positions, 160 rows stay with the kernel for few."""
    f = Filled([150, 37], 2, 128, 128, E4M3, 64, seed=24, table_pages=32768)
    q = rand_q(2, 40, 8, 128)
    free = torch.cuda.mem_get_info()[0]
    a = check_attention(f, q)
    assert free - torch.cuda.mem_get_info()[0] < 1 << 30
    b = check_attention(f, q, max_seqlen=150)
    assert torch.allclose(a[0].float(), b[0].float(), rtol=2e-2, atol=2e-2)
    odd = torch.zeros(2, 40, 8, 129, dtype=torch.bfloat16, device="cuda")[..., 1:]          # rows that 16-byte vectors cannot read
    odd.copy_(q)
    c = fm.kv_cache_attention(odd, f.cache, f.table.cuda(), f.seqlens.cuda(), max_seqlen=150)
    assert torch.equal(b[0], c)


def test_long_cache_many_parts():
    """More units than CTAs, so that items are cut in every place."""
    f = Filled([5000, 3, 1300, 2049], 2, 64, 64, E4M3, 128, seed=12)
    check_attention(f, rand_q(4, 1, 8, 64))
    f = Filled([9000], 1, 128, 128, INT8, 64, seed=13)
    check_attention(f, rand_q(1, 3, 4, 128), window=4000)


def test_many_sequences():
    """More sequences than threads of a CTA."""
    lens = [(i * 37) % 50 for i in range(600)]
    f = Filled(lens, 1, 16, 16, INT8, 16, seed=14)
    check_attention(f, rand_q(600, 1, 2, 16))


def test_large_scores_and_scales():
    """Scores that grow along the sequence (the lagging maximum has to move), queries at the ends of bf16's range."""
    f = Filled([400], 1, 64, 64, E4M3, 16, seed=15)
    q = rand_q(1, 2, 4, 64, size=30.0)
    check_attention(f, q)
    q = rand_q(1, 1, 4, 64)
    q[0, 0, 0] *= 2.0 ** 100
    q[0, 0, 1] *= 2.0 ** -100
    check_attention(f, q[:, :, 1:], scale=0.125)
    f.cache.k_scale.mul_(2.0 ** -60)
    check_attention(f, q[:, :, :1], scale=2.0 ** -42)
    f.cache.v_scale[::2] *= 2.0 ** 40
    check_attention(f, q[:, :, 1:2])


@pytest.mark.parametrize("d,dv,S", [(192, 128, 130), (192, 128, 230), (256, 256, 32), (256, 256, 40)])
def test_many_rows_of_wide_heads(d, dv, S):
    """Rows on both sides of where the dense forward takes over (three sequences of 2 kv heads: 900 rows | 150 rows)."""
    f = Filled([300, 37, 150], 2, d, dv, E4M3, 32, seed=25)
    check_attention(f, rand_q(3, S, 8, d, seed=26), q_lengths=[S, 20, S - 9])
    check_attention(f, rand_q(3, S, 8, d, seed=27), causal=False)


@pytest.mark.parametrize("d,G", [(64, 1), (64, 9), (128, 2)])
def test_as_many_sequences_as_a_call_takes(d, G):
    """1024 short ones and a long one among them, which is cut."""
    lens = [(i * 29) % 40 for i in range(1024)]
    lens[500] = 1500
    f = Filled(lens, 1, d, d, E4M3, 16, seed=23)
    check_attention(f, rand_q(1024, 1, G, d, seed=24))


@pytest.mark.parametrize("kind", [E4M3, INT8])
@pytest.mark.parametrize("S,window", [(1, None), (3, None), (3, 24)])
def test_nan_where_nobody_looks(kind, S, window):
    """NaN in slots behind the sequence, in pages of others, in front of the window, and in tokens that only later rows see."""
    f = Filled([45, 33], 1, 64, 64, kind, 16, seed=16)
    q = rand_q(2, S, 4, 64)
    clean = fm.kv_cache_attention(q.cuda(), f.cache, f.table.cuda(), f.seqlens.cuda(), window_size=window, return_lse=True)
    nan = 0x7f if kind == E4M3 else 0x80
    owned = set(f.table.flatten().tolist())
    for name in "kv":
        raw = getattr(f.cache, name).view(torch.uint8)
        for b in range(2):
            raw[f.table[b, f.lens[b] // 16], :, f.lens[b] % 16:] = nan
        for p in set(range(raw.shape[0])) - owned:
            raw[p] = nan
            getattr(f.cache, name + "_scale")[p] = math.nan
        if window:
            raw[f.table[0, 0]] = nan
    dirty = fm.kv_cache_attention(q.cuda(), f.cache, f.table.cuda(), f.seqlens.cuda(), window_size=window, return_lse=True)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    if S == 3:
        # the last token's value (key) is NaN: the rows before it stay as they were, its own becomes NaN
        if kind == E4M3:
            f.cache.v.view(torch.uint8)[f.table[0, 2], 0, 44 % 16, 7] = 0xff
            out = fm.kv_cache_attention(q.cuda(), f.cache, f.table.cuda(), f.seqlens.cuda(), window_size=window)
            assert torch.equal(out[0, :2], clean[0][0, :2]) and torch.equal(out[1], clean[0][1])
            want = torch.zeros(64, dtype=torch.bool)
            want[7] = True
            assert torch.equal(torch.isnan(out[0, 2]).cpu(), want.expand(4, 64))
            f.cache.k.view(torch.uint8)[f.table[0, 2], 0, 44 % 16, 7] = 0xff
            out = fm.kv_cache_attention(q.cuda(), f.cache, f.table.cuda(), f.seqlens.cuda(), window_size=window)
            assert torch.equal(out[0, :2], clean[0][0, :2]) and torch.isnan(out[0, 2]).all()


def test_bad_pages_are_no_tokens():
    f = Filled([100, 60], 2, 64, 64, E4M3, 16, seed=17)
    f.table[0, 1], f.table[0, 4], f.table[1, 0] = -1, f.cache.k.shape[0], 2 ** 31 - 1
    check_attention(f, rand_q(2, 2, 8, 64))
    check_attention(f, rand_q(2, 40, 8, 64))
    f.lens = [10 ** 6, -3]                              # beyond the page table, and below nothing
    f.seqlens = torch.tensor(f.lens, dtype=torch.int32)
    check_attention(f, rand_q(2, 2, 8, 64))


def test_shared_prefix_pages_and_strided_table():
    f = Filled([64, 64], 2, 64, 64, E4M3, 16, seed=18)
    f.table[1, :2] = f.table[0, :2]
    q = rand_q(2, 1, 8, 64)
    a = check_attention(f, q)
    wide = torch.full((2, 9), -7, dtype=torch.int32)
    wide[:, 2:6] = f.table
    b = fm.kv_cache_attention(q.cuda(), f.cache, wide.cuda()[:, 2:6], f.seqlens.cuda(), return_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    qs = torch.zeros(2, 1, 24, 64, dtype=torch.bfloat16)
    qs[:, :, 8:16] = q
    c = fm.kv_cache_attention(qs.cuda()[:, :, 8:16], f.cache, f.table.cuda(), f.seqlens.cuda())
    assert torch.equal(a[0], c)


def test_empty_calls():
    f = Filled([5], 1, 32, 32, E4M3, 16, seed=19)
    t = f.table.cuda()
    out, lse = fm.kv_cache_attention(torch.zeros(0, 1, 2, 32, dtype=torch.bfloat16, device="cuda"), f.cache, t[:0], f.seqlens.cuda()[:0], return_lse=True)
    assert out.shape == (0, 1, 2, 32) and lse.shape == (0, 2, 1)
    out, lse = fm.kv_cache_attention(torch.zeros(1, 0, 2, 32, dtype=torch.bfloat16, device="cuda"), f.cache, t, f.seqlens.cuda(), return_lse=True)
    assert out.shape == (1, 0, 2, 32) and lse.shape == (1, 2, 0)
    out, lse = fm.kv_cache_attention(rand_q(1, 1, 2, 32).cuda(), f.cache, t[:, :0], f.seqlens.cuda(), return_lse=True)
    assert not out.any() and torch.isinf(lse).all()
    k, v = fm.kv_cache_read(f.cache, t, f.seqlens.cuda(), f.seqlens.cuda(), 0)
    assert k.shape == (1, 0, 1, 32)
    fm.kv_cache_write(f.cache, k, v, t, f.seqlens.cuda())


def test_same_bits_on_every_call_and_on_another_stream():
    f = Filled([3000, 700], 2, 128, 128, E4M3, 64, seed=20)
    q, t, n = rand_q(2, 1, 8, 128).cuda(), f.table.cuda(), f.seqlens.cuda()
    a = fm.kv_cache_attention(q, f.cache, t, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = [fm.kv_cache_attention(q, f.cache, t, n) for _ in range(5)]
    c = [fm.kv_cache_attention(q, f.cache, t, n) for _ in range(5)]
    torch.cuda.synchronize()
    for x in b + c:
        assert torch.equal(a, x)


def test_refusals():
    f = Filled([20], 2, 64, 64, E4M3, 16, seed=21)
    q, t, n = rand_q(1, 1, 4, 64).cuda(), f.table.cuda(), f.seqlens.cuda()
    call = lambda q=q, c=f.cache, t=t, n=n, **kw: fm.kv_cache_attention(q, c, t, n, **kw)
    call()
    for bad in (dict(q=q[..., :32]), dict(q=q[:, :, :3]), dict(t=t.long()), dict(t=t.cpu()), dict(n=n.long()), dict(n=n[:0]), dict(sink=torch.zeros(3).cuda())):
        with pytest.raises(AssertionError):
            call(**bad)
    with pytest.raises(TypeError):
        call(q=q.float())
    with pytest.raises(RuntimeError):
        call(q=q.cpu())
    with pytest.raises(RuntimeError, match="no gradient"):
        call(q=q.clone().requires_grad_(True))
    with pytest.raises(ValueError):
        call(causal=False, window_size=4)
    with pytest.raises(ValueError):
        call(window_size=0)
    k = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(AssertionError):
        fm.kv_cache_write(f.cache, k[:, :, :1], k[:, :, :1], t, n)
    with pytest.raises(AssertionError):
        fm.kv_cache_write(f.cache, k, k.half(), t, n)
    odd = fm.QuantizedKVCache(*(torch.zeros(2, 2, 48, 64, dtype=torch.int8, device="cuda") for _ in range(2)),
                              *(torch.ones(2, 2, device="cuda") for _ in range(2)))
    with pytest.raises(NotImplementedError):
        call(c=odd)
    mixed = fm.QuantizedKVCache(f.cache.k, f.cache.v.view(torch.int8), f.cache.k_scale, f.cache.v_scale)
    with pytest.raises(AssertionError):
        call(c=mixed)


def test_generation_replays_from_a_cuda_graph():
    """Norm and rotation, append, attention, captured once and replayed with lengths that grow on the device: the bits of
    the eager steps."""
    B, H, G, d, page, steps = 2, 2, 4, 64, 16, 20
    g = torch.Generator().manual_seed(22)
    xs = torch.randn(steps, B, 1, H * G + 2 * H, d, generator=g).bfloat16().cuda()
    w = [torch.randn(d, generator=g).bfloat16().cuda() for _ in range(2)]
    angle = torch.arange(64)[:, None] * 10000.0 ** (-torch.arange(d // 2) / (d // 2))[None]
    cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()
    table = torch.tensor([[0, 1, 2], [5, 4, 3]], dtype=torch.int32).cuda()

    def step(x, cache, start):
        q, k = fm.qk_norm_rotary(x[:, :, :H * G], x[:, :, H * G:H * G + H], *w, cos, sin, start.view(B, 1))
        fm.kv_cache_write(cache, k, x[:, :, H * G + H:], table, start)
        return fm.kv_cache_attention(q, cache, table, start + 1, return_lse=True)

    eager, cache = [], fm.QuantizedKVCache.empty(6, H, d, page_size=page)
    start = torch.tensor([0, 11], dtype=torch.int32).cuda()
    with torch.no_grad():
        for i in range(steps):
            eager.append([t.clone() for t in step(xs[i], cache, start + i)])
        cache2, x, at = fm.QuantizedKVCache.empty(6, H, d, page_size=page), xs[0].clone(), start.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, cache2, at)
        torch.cuda.current_stream().wait_stream(side)
        cache2 = fm.QuantizedKVCache.empty(6, H, d, page_size=page)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(x, cache2, at)
        for i in range(steps):
            x.copy_(xs[i])
            at.copy_(start + i)
            graph.replay()
            for a, b in zip(got, eager[i]):
                assert torch.equal(a, b), i
    for n in "kv":
        assert torch.equal(getattr(cache, n).view(torch.uint8), getattr(cache2, n).view(torch.uint8))


def test_two_graphs_and_two_streams_share_nothing():
    """Two captured calls replayed in turn and against each other on two streams, one with many parts, one through the dense forward."""
    f, g = Filled([3000, 900], 2, 128, 128, E4M3, 64, seed=25), Filled([700, 333], 2, 128, 128, INT8, 32, seed=26)
    q1, q2 = rand_q(2, 1, 8, 128).cuda(), rand_q(2, 40, 8, 128, seed=2).cuda()
    args = [(q1, f.cache, f.table.cuda(), f.seqlens.cuda()), (q2, g.cache, g.table.cuda(), g.seqlens.cuda())]
    want = [fm.kv_cache_attention(*a, return_lse=True) for a in args]
    graphs, got = [], []
    for a in args:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(fm.kv_cache_attention(*a, return_lse=True))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for x in got:
            for t in x:
                t.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager = []
        for a, s in zip(args, streams):
            with torch.cuda.stream(s):
                eager.append(fm.kv_cache_attention(*a, return_lse=True))
        torch.cuda.synchronize()
        for w, x, y in zip(want, got, eager):
            for a, b, c in zip(w, x, y):
                assert torch.equal(a, b) and torch.equal(a, c)


def test_prompt_then_tokens_is_attention_over_everything():
    """A prompt written and attended to in one call, then token by token: every step against the dense operator over what
    the cache gives back, within the rounding of p and of the output."""
    H, G, d, page, S = 2, 4, 128, 64, 150
    g = torch.Generator().manual_seed(23)
    qs, ks, vs = (torch.randn(1, S, h, d, generator=g).bfloat16().cuda() for h in (H * G, H, H))
    cache = fm.QuantizedKVCache.empty(4, H, d, page_size=page)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32).cuda()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()
    outs, at = [], 0
    for n in (140, 1, 1, 5, 3):
        fm.kv_cache_write(cache, ks[:, at:at + n], vs[:, at:at + n], table, i32(at))
        outs.append(fm.kv_cache_attention(qs[:, at:at + n], cache, table, i32(at + n)))
        at += n
    k, v = fm.kv_cache_read(cache, table, i32(0), i32(S), S)
    for n, out, end in ((3, outs[-1], 150), (5, outs[-2], 147)):
        want = fm.flashmask_attention(qs[:, end - n:end], k[:, :end], v[:, :end], causal=True)
        weight = fm.flashmask_attention(qs[:, end - n:end], k[:, :end], v[:, :end].abs(), causal=True)
        # half steps: p on one side 2^-8, on the other 2^-11, the results 2^-8 each, and the weight itself 2^-8
        assert ((out.float() - want.float()).abs() <= (3 * 2.0 ** -8 + 2.0 ** -10) * 1.01 * weight.float() + 1e-6).all()
