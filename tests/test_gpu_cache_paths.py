"""Attention over the cache on both of its paths, the kernel that reads pages and the dense forward over tokens read back, where a
call can go wrong: NaN that a row does not see, windows and page tables of any width, many K tiles under a mask, wide heads."""
import math

import pytest
import torch

import flashmask_b200 as fm
import _cache_util as ref
from test_gpu_cache import E4M3, INT8, Filled, rand_q

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def defined(q, k, v, there, n_rows, causal, window, scale, sink):
    """One sequence in 64 bits: out [S, Hq, dv], lse [Hq, S], and for the tolerances sum_j p_j |v_j| and the largest sum_c |q_c k_c| of a
    visible key [S, Hq].  NaN in a key or value reaches the rows that see it."""
    S, Hq, d = q.shape
    L, H = k.shape[:2]
    at = (torch.arange(S, device="cuda") + L - n_rows)[:, None]
    pos = torch.arange(L, device="cuda")[None]
    seen = there[None] & ((pos <= at) if causal else torch.ones_like(pos <= at)) & (torch.arange(S, device="cuda") < n_rows)[:, None]
    if window:
        seen = seen & (pos > at - window)
    out, weight = (torch.zeros(S, Hq, v.shape[2], dtype=torch.float64, device="cuda") for _ in range(2))
    lse, reach = torch.full((Hq, S), -math.inf, dtype=torch.float64, device="cuda"), torch.zeros(S, Hq, dtype=torch.float64, device="cuda")
    some = seen.any(1)
    for h in range(Hq):
        kk, vv = k[:, h * H // Hq], v[:, h * H // Hq]
        x = torch.where(seen, q[:, h] @ kk.T * scale, torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
        if sink is not None:
            x = torch.cat([x, sink[h].double().cuda().expand(S, 1)], 1)
        lse[h] = torch.logsumexp(x, 1)
        p = torch.where(seen, torch.softmax(x, 1)[:, :L], torch.zeros((), dtype=torch.float64, device="cuda"))
        out[:, h] = p @ vv.nan_to_num(nan=0.0)
        out[:, h][(seen.double() @ vv.isnan().double()) > 0] = math.nan
        out[~some, h] = 0.0
        weight[:, h] = p @ vv.abs().nan_to_num(nan=0.0)
        reach[:, h] = torch.where(seen, q[:, h].abs() @ kk.abs().T, torch.zeros((), dtype=torch.float64, device="cuda")).amax(1) * abs(scale) if L else 0.0
    return [t.cpu() for t in (out, lse, weight, reach)]


def agrees(f, q, pages, *, q_lengths=None, causal=True, window=None, scale=None, sink=None, **kw):
    """The call against the definition.  `pages`: the kernel that reads pages takes it (p in fp16), else the dense forward (p in
    q's type).  Where the definition has NaN the result has, and nowhere else; its lse is NaN where a whole row is.

    Half a step of p is 2^-11 in fp16 and 2^-8 in bf16; in fp16 it is absolute below 2^-14: 2^-25, when the largest p is 2^7 at
    least (pages) or 1 (dense), of values of at most 448 scales.  A score is off by d + 16 steps of 2^-23 of the sum of its
    products' magnitudes, a sum over n keys by n steps of 2^-24, and the result is rounded once.  A sink far above the scores makes
    the denominator up to 2^127, whose reciprocal is flushed to 0 below 2^-126: that takes at most 2^-126 of the row's sum before the
    division, n weights of at most 2^15 (pages) or 2^8 (dense) of those values, 2^-111 n 448 scales."""
    B, S, Hq, d = q.shape
    got = fm.kv_cache_attention(q.cuda(), f.cache, f.table.cuda(), f.seqlens.cuda(), causal=causal, window_size=window,
                                q_lengths=None if q_lengths is None else i32(q_lengths), softmax_scale=scale,
                                sink=None if sink is None else sink.cuda(), return_lse=True, **kw)
    out, lse = got[0].cpu().double(), got[1].cpu().double()
    half = torch.finfo(q.dtype).eps / 2
    p_half, p_least = (2.0 ** -11, 2.0 ** -32) if pages else ((2.0 ** -11, 2.0 ** -25) if q.dtype == FP16 else (2.0 ** -8, 0.0))
    for b in range(B):
        n = min(max(f.lens[b], 0), f.table.shape[1] * f.page)
        (k, there), (v, _) = f.dense(b, "k", n), f.dense(b, "v", n)
        rows = S if q_lengths is None else min(max(q_lengths[b], 0), S)
        o, l, weight, reach = defined(q[b].double().cuda(), k.cuda(), v.cuda(), there.cuda(), rows, causal, window, 1 / math.sqrt(d) if scale is None else scale, sink)
        assert torch.equal(torch.isnan(out[b]), torch.isnan(o)), b
        dead = torch.isnan(o).all(-1)
        assert torch.equal(torch.isnan(lse[b]), dead.T), b
        slack = reach * (d + 16) * 2.0 ** -23 + 2.0 ** -20 + max(n, 1) * 2.0 ** -24
        tol = half * o.abs() + n * p_least * 448 * f.largest_scale(b) + weight * (p_half + 2 * slack[..., None]) + torch.finfo(q.dtype).smallest_normal * half
        if sink is not None:
            tol = tol + n * 2.0 ** -111 * 448 * f.largest_scale(b)
        far = ((out[b] - o).abs() - tol).nan_to_num(nan=-1.0)
        w = far.argmax()
        assert far.flatten()[w] <= 0, (b, int(w), *(t.flatten()[w].item() for t in (far, out[b], o, weight)))
        fin = torch.isfinite(l) & ~dead.T
        assert torch.equal(torch.isinf(lse[b]) | dead.T, ~fin), b
        ltol = (slack.T + 2.0 ** -21 * l.abs())[fin] + 2.0 ** -20
        assert ((lse[b] - l).abs()[fin] <= ltol).all(), (b, (lse[b] - l).abs()[fin].max())
    return got


def page_at(f, b, pos):
    return int(f.table[b, pos // f.page])


def plant(f, S):
    """NaN in a value in the middle of the queries' own tokens (head 0), in a key near the end and in a value at the start (last head).  In int8
    it is the page's scale that says so, and the whole page that is none."""
    last = f.cache.k.shape[1] - 1
    for b, n in enumerate(f.lens):
        for name, pos, h, dim in (("v", n - S // 2, 0, 7), ("k", n - 3, last, 5), ("v", 3, last, 1)):
            if pos < 0:
                continue
            page = page_at(f, b, pos)
            if f.kind == E4M3:
                getattr(f.cache, name).view(torch.uint8)[page, h, pos % f.page, dim] = 0xff if dim == 7 else 0x7f
            else:
                getattr(f.cache, name + "_scale")[page, h] = math.nan


MASKS = [(True, None, False), (True, 33, True), (False, None, True)]


@pytest.mark.parametrize("kind", [E4M3, INT8])
@pytest.mark.parametrize("causal,window,padded", MASKS)
@pytest.mark.parametrize("S,G,d,dv,dtype,pages", [(20, 4, 128, 128, BF16, True), (40, 4, 128, 128, BF16, False), (40, 3, 64, 64, FP16, False), (120, 1, 80, 48, BF16, False),
                                                  (40, 4, 192, 128, BF16, True), (40, 4, 256, 256, BF16, False), (20, 4, 256, 256, FP16, True)])
def test_nan_reaches_the_rows_that_see_it_alone(kind, causal, window, padded, S, G, d, dv, dtype, pages):
    f = Filled([300, 37, 170], 2, d, dv, kind, 16, seed=31, dtype=dtype)
    plant(f, S)
    agrees(f, rand_q(3, S, 2 * G, d, seed=32, dtype=dtype), pages, causal=causal, window=window, q_lengths=[S, 11, S - 9] if padded else None)


@pytest.mark.parametrize("kind", [E4M3, INT8])
@pytest.mark.parametrize("S,G,d,dv,dtype", [(32, 4, 64, 64, FP16), (100, 4, 128, 128, BF16), (230, 4, 192, 128, BF16), (300, 2, 128, 64, FP16)])
def test_nan_in_a_long_prompt_in_parts(kind, S, G, d, dv, dtype):
    """Many K tiles, dealt to several CTAs; queries of several row blocks; a sink; NaN queries of rows that see something."""
    f = Filled([2900, 500, 1000], 2, d, dv, kind, 64, seed=33, dtype=dtype)
    plant(f, S)
    q = rand_q(3, S, 2 * G, d, seed=34, dtype=dtype)
    agrees(f, q, False, sink=torch.linspace(-1, 2, 2 * G))
    agrees(f, q, False, window=700)
    clean = Filled([2900, 500, 1000], 2, d, dv, kind, 64, seed=33, dtype=dtype)
    q[1, 5, 1, 3] = math.nan
    agrees(clean, q, False)


@pytest.mark.parametrize("kind", [E4M3, INT8])
def test_many_rows_that_see_no_nan_keep_their_bits(kind):
    """Slots behind the sequences, pages of others, tokens in front of the window, tokens that only later rows see."""
    S = 40
    f, g = (Filled([300, 45], 2, 64, 64, kind, 16, seed=35) for _ in range(2))
    q = rand_q(2, S, 8, 64, seed=36)
    nan = 0x7f if kind == E4M3 else 0x80
    owned = set(f.table.flatten().tolist())
    for name in "kv":
        raw = getattr(g.cache, name).view(torch.uint8)
        for b in range(2):
            raw[page_at(g, b, g.lens[b]), :, g.lens[b] % 16:] = nan
        for p in set(range(raw.shape[0])) - owned:
            raw[p] = nan
            getattr(g.cache, name + "_scale")[p] = math.nan
        getattr(g.cache, name + "_scale")[page_at(g, 0, 200)] = math.nan              # positions 192 .. 207: in front of the window
    a, b = (agrees(x, q, False, window=30) for x in (f, g))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    if kind == E4M3:
        g.cache.v.view(torch.uint8)[page_at(g, 0, 290), 1, 290 % 16, 9] = 0xff
        c = agrees(g, q, False, window=30)
        seen = torch.zeros(2, S, 8, 64, dtype=torch.bool)
        seen[0, 30:, 4:, 9] = True                                                  # rows from position 290 on, whose windows hold it
        assert torch.equal(torch.isnan(c[0]).cpu(), seen) and torch.equal(c[0][~seen.cuda()], a[0][~seen.cuda()]) and torch.equal(c[1], a[1])


@pytest.mark.parametrize("d,dv,S,H", [(64, 64, 40, 2), (128, 128, 40, 1), (192, 128, 340, 2)])
@pytest.mark.parametrize("bound", [None, 300000])
def test_more_positions_than_the_dense_forward_takes(d, dv, S, H, bound):
    """A page table, or an upper bound, of 300000 positions over short sequences: 262144 are the most that the dense forward takes."""
    f = Filled([400, 37], H, d, dv, E4M3, 128, seed=37, table_pages=2344)
    agrees(f, rand_q(2, S, 4 * H, d, seed=38), True, max_seqlen=bound)


@pytest.mark.parametrize("window", [1, 64, 1000])
@pytest.mark.parametrize("padded", [False, True])
def test_a_window_bounds_what_is_read_back(window, padded):
    """A window far below the length, with and without an upper bound; a page table whose dense tensors would take 2 GiB without a
    window takes a few MiB."""
    f = Filled([5000, 37, 1200], 2, 64, 64, E4M3, 64, seed=39, table_pages=4096)
    q = rand_q(3, 40, 8, 64, seed=40)
    kw = dict(window=window, q_lengths=[40, 11, 25] if padded else None)
    a = agrees(f, q, False, **kw)
    b = agrees(f, q, False, max_seqlen=5000, **kw)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    args = (q.cuda(), f.cache, f.table.cuda(), f.seqlens.cuda())
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    fm.kv_cache_attention(*args, window_size=window)
    # the dense tensors: 1039 columns of 3 sequences, 2 heads, 64 + 64 values of 2 bytes, 1.6 MB; out, lse, bounds and partial results beside them
    assert torch.cuda.max_memory_allocated() - before < 16 << 20
    # more tokens than the dense forward takes, of which the window leaves few
    g = Filled([5000, 37, 1200], 2, 64, 64, E4M3, 64, seed=39, table_pages=5000)
    c = agrees(g, q, False, **kw)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


@pytest.mark.parametrize("d,dv,dtype", [(64, 64, FP16), (80, 80, BF16), (96, 96, FP16), (96, 128, BF16), (112, 16, BF16), (128, 128, BF16)])
@pytest.mark.parametrize("S,G,window,causal", [(32, 4, None, True), (100, 1, 700, True), (64, 4, None, False), (40, 3, 2000, True), (300, 4, 1500, True)])
def test_many_tiles_under_a_mask(d, dv, dtype, S, G, window, causal):
    """The dense forward's deal of K tiles to CTAs and sub-tiles when a mask tensor is there: parts that lengths and windows leave
    empty, one row block (sub-tiles in turn) and several, packed heads and not, rows that see nothing."""
    f = Filled([4100, 37, 700], 2, d, dv, E4M3, 64, seed=41, dtype=dtype)
    q = rand_q(3, S, 2 * G, d, seed=42, dtype=dtype)
    agrees(f, q, False, window=window, causal=causal)
    agrees(f, q, False, window=window, causal=causal, q_lengths=[S, 0, S // 2], sink=torch.linspace(-2, 2, 2 * G))


@pytest.mark.parametrize("d,dv,S", [(192, 128, 130), (192, 128, 225), (256, 256, 30)])
@pytest.mark.parametrize("kind", [E4M3, INT8])
def test_wide_heads_with_many_rows_keep_the_precision_of_pages(d, dv, S, kind):
    """Three sequences of two kv heads: up to 900 | 150 rows stay with the kernel that reads pages, whose p is fp16 whatever q is."""
    f = Filled([300, 37, 150], 2, d, dv, kind, 32, seed=43)
    agrees(f, rand_q(3, S, 8, d, seed=44), True, q_lengths=[S, 20, S - 9])


@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_scales_that_turn_scores_round(scale):
    f = Filled([300, 37], 2, 64, 64, E4M3, 16, seed=45)
    for S, pages in ((3, True), (40, False)):
        agrees(f, rand_q(2, S, 8, 64, seed=46), pages, scale=scale, window=50)


def test_positions_at_the_end_of_a_table_of_two_billion():
    """A write of 70000 rows, of which five count, that starts near the end of a page table of 2^31 - 2^16 - 128 positions; and one that
    runs over that end."""
    page, n = 128, (2 ** 31 - 2 ** 16) // 128 - 1
    table = torch.full((1, n), -1, dtype=torch.int32, device="cuda")
    table[0, n - 1], table[0, n - 2] = 1, 0
    x = torch.randn(1, 70000, 1, 16, generator=torch.Generator().manual_seed(47)).bfloat16().cuda()
    for start, rows in ((n * page - page - 2, 5), (n * page - 4, 70000)):
        cache = fm.QuantizedKVCache.empty(2, 1, 16, page_size=page)
        fm.kv_cache_write(cache, x, x, table, i32([start]), i32([rows]))
        want = fm.QuantizedKVCache.empty(2, 1, 16, page_size=page)
        at = start - (n - 2) * page                                                 # the same slots through a table of two pages
        fm.kv_cache_write(want, x[:, :256].contiguous(), x[:, :256].contiguous(), i32([[0, 1]]), i32([at]), i32([min(rows, 256)]))
        assert want.k.view(torch.uint8).any()
        for a in ("k", "v", "k_scale", "v_scale"):
            assert torch.equal(getattr(cache, a).view(torch.uint8), getattr(want, a).view(torch.uint8)), (a, start)


@pytest.mark.parametrize("kind", [E4M3, INT8])
def test_appends_that_grow_the_scale_of_pages_that_warps_take(kind):
    """A token appended to each of 256 pages of 8 heads, 4096 warps side by side, each token larger than those before: the earlier
    tokens are rounded again from the scale that the page had."""
    B, H, d, page = 256, 8, 32, 16
    cache = fm.QuantizedKVCache.empty(B, H, d, page_size=page, dtype=kind)
    table = torch.randperm(B, generator=torch.Generator().manual_seed(48)).int()[:, None]
    vals = {n: getattr(cache, n).cpu().float().double()[:4] for n in "kv"}
    where = [int((table[:, 0] == p).nonzero()) for p in range(4)]                  # sequences of the pages that the oracle follows
    sc = {n: getattr(cache, n + "_scale").cpu().double()[:4] for n in "kv"}
    g = torch.Generator().manual_seed(49)
    for step in range(6):
        x = {n: (torch.randn(B, 1, H, d, generator=g) * 3.0 ** step).bfloat16() for n in "kv"}
        fm.kv_cache_write(cache, x["k"].cuda(), x["v"].cuda(), table.cuda(), i32([step] * B))
        for n in "kv":
            ref.write((vals[n], kind), sc[n], x[n][where], torch.arange(4).int()[:, None], [step] * 4, None)
    for n in "kv":
        assert torch.equal(getattr(cache, n + "_scale").cpu().double()[:4], sc[n])
        assert torch.equal(getattr(cache, n).cpu().float().double()[:4], vals[n])


def test_tangents_are_refused():
    """No operator of the cache has a derivative: a dual tensor is refused, under no_grad too, and not taken for a constant."""
    import torch.autograd.forward_ad as ad
    f = Filled([20], 2, 64, 64, E4M3, 16, seed=50)
    q, t, n = rand_q(1, 1, 4, 64).cuda(), f.table.cuda(), f.seqlens.cuda()
    k = torch.ones(1, 1, 2, 64, dtype=BF16, device="cuda")
    sink = torch.zeros(4, device="cuda")
    with ad.dual_level():
        dual = lambda x: ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: fm.kv_cache_attention(dual(q), f.cache, t, n), lambda: fm.kv_cache_attention(q, f.cache, t, n, sink=dual(sink)),
                     lambda: fm.kv_cache_write(f.cache, dual(k), k, t, n), lambda: fm.kv_cache_write(f.cache, k, dual(k), t, n)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
                call()
        fm.kv_cache_attention(q, f.cache, t, n, sink=sink)


def test_caches_that_want_a_gradient_are_refused():
    f = Filled([20], 2, 64, 64, E4M3, 16, seed=51)
    t, n = f.table.cuda(), f.seqlens.cuda()
    k = torch.ones(1, 1, 2, 64, dtype=BF16, device="cuda")
    for name in ("k_scale", "v_scale"):
        getattr(f.cache, name).requires_grad_(True)
        for call in (lambda: fm.kv_cache_attention(rand_q(1, 1, 4, 64).cuda(), f.cache, t, n), lambda: fm.kv_cache_read(f.cache, t, n - 5, n, 5),
                     lambda: fm.kv_cache_write(f.cache, k, k, t, n)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
            with torch.no_grad():
                call()
        getattr(f.cache, name).requires_grad_(False)


@pytest.mark.parametrize("S,G,d,dv,dtype,pages", [(5, 4, 128, 128, BF16, True), (40, 4, 64, 64, FP16, False), (140, 1, 128, 128, BF16, False), (300, 3, 128, 128, BF16, False),
                                                  (240, 4, 192, 128, BF16, False), (60, 4, 256, 256, BF16, False), (300, 4, 256, 256, FP16, False)])
@pytest.mark.parametrize("scale", [None, -0.1])
def test_sinks_far_from_every_score(S, G, d, dv, dtype, pages, scale):
    """A sink that is all there is to a row, its scores 2^127 below it and more, and one that is small beside nothing: rows that see nothing."""
    f = Filled([2000, 300, 0, 20], 2, d, dv, E4M3, 64, seed=52, dtype=dtype)
    sink = torch.tensor([200.0, -200.0, 0.5, -95.0, 95.0, -1e4])[torch.arange(2 * G) % 6]
    out, lse = agrees(f, rand_q(4, S, 2 * G, d, seed=53, dtype=dtype), pages, sink=sink, scale=scale, q_lengths=[S, S // 2, S, S])
    assert torch.equal(lse[2], sink[:, None].expand(2 * G, S).cuda())


def test_a_captured_chunk_sees_what_the_cache_holds_at_a_replay():
    """NaN that comes and goes between replays, and lengths that change: every replay gives the bits of an eager call."""
    f = Filled([300, 170], 2, 64, 64, E4M3, 16, seed=54)
    q, table, n = rand_q(2, 40, 8, 64, seed=55).cuda(), f.table.cuda(), f.seqlens.cuda()
    clean = f.cache.v.view(torch.uint8).clone()
    call = lambda: fm.kv_cache_attention(q, f.cache, table, n, max_seqlen=300, return_lse=True)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for pos, lens in ((280, [300, 170]), (None, [300, 170]), (130, [290, 120]), (130, [290, 160])):
        f.cache.v.view(torch.uint8).copy_(clean)
        n.copy_(torch.tensor(lens))
        if pos is not None:
            for b in range(2):
                f.cache.v.view(torch.uint8)[page_at(f, b, min(pos, 160)), 1, pos % 16, 3] = 0x7f
        graph.replay()
        for a, b in zip(got, call()):
            assert torch.equal(a.nan_to_num(nan=77.0), b.nan_to_num(nan=77.0))
        assert bool(torch.isnan(got[0]).any()) == (pos is not None)
