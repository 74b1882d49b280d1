"""GPU: the paged key/value cache against plain 64-bit loops: write, attention of one token, eviction, and the three in turn.

Tolerance of attention.  A row's score is a dot product of D terms in fp32 (off by (D + 4) 2^-24 of ``sum |q_d k_d|``, here
``dots`` in natural units; the tensor cores may cut sums to 2^-22 instead of rounding them, so (D + 4) 2^-22), its exponential
by 2^-21 beyond that, the sums of n terms by n 2^-24 at most.  So a weight is off by ``rel = 2 dots (D + 4) 2^-22 + 2^-20 + n 2^-23``
of itself, an output by that of ``sum p |v|`` (``mass``).  Where the tensor cores multiply 16-bit weights, ``o = sum p' v / sum p'`` with every ``p'``
half a step off at most: half a step of ``mass`` from the numerator and half a step of ``o`` from the denominator.  Then ``o`` is rounded,
by half a step again.
"""

import pytest
import torch

from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu

F32, F16, BF16, F8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _to(x, dtype):
    return x.clamp(-448, 448).to(dtype) if dtype == F8 else x.to(dtype)


def make_cache(B, H_kv, D, page, lens, dtype, seed=0, spare=3, M=None, stale=None):
    """CPU tensors of a cache in use: pages handed out in any order, entries behind a sequence's last page point nowhere."""
    g = torch.Generator().manual_seed(seed)
    lens = torch.tensor(lens, dtype=torch.int32)
    need = [-(-max(int(n), 0) // page) for n in lens]
    M = max(need + [1]) if M is None else M
    P = sum(need) + spare
    order, table = torch.randperm(P, generator=g).tolist(), torch.full((B, M), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    table[table < 0] = torch.tensor([-1, P, 2**31 - 1, -2**31])[torch.arange(int((table < 0).sum())) % 4].to(torch.int32)
    c = dict(page_table=table, lens=lens)
    for n in ("k", "v"):
        x = torch.randn(P, H_kv, page, D, generator=g)
        c[n + "_pages"] = _to(x * 100, F8) if dtype == F8 else x.to(dtype)
        if dtype == F8:
            c[n + "_scale"] = torch.rand(P, H_kv, page, generator=g) * 0.01 + 0.005
    if stale is not None:  # rows that belong to nobody
        used = torch.zeros(P, page, dtype=torch.bool)
        for b, n in enumerate(lens.tolist()):
            for r in range(max(n, 0)):
                used[table[b, r // page], r % page] = True
        for n in ("k", "v"):
            bytes_ = c[n + "_pages"]
            bytes_.view(torch.uint8)[~used[:, None].expand(P, H_kv, page)] = torch.full((1, D), stale, dtype=F32).to(dtype).view(torch.uint8)
            if dtype == F8:
                c[n + "_scale"][~used[:, None].expand(P, H_kv, page)] = stale
    return c


def cuda(c):
    return {n: x.cuda() for n, x in c.items()}


def check_attend(c, q, context_size=None, back=0, sm_scale=None, weights=None, on_gpu=None, **more):
    from kernels_b200.streaming_attention import paged_attention

    B, H, D = q.shape
    H_kv = c["k_pages"].shape[1]
    group = H // H_kv
    ref_o, ref_lse, ref_w, (dots, mass) = PO.attend(q, c["k_pages"], c["v_pages"], c["page_table"], c["lens"], context_size, back, sm_scale,
                                                    c.get("k_scale"), c.get("v_scale"))
    g = cuda(c) if on_gpu is None else on_gpu
    w = None if weights is None else weights.cuda()
    o, lse = paged_attention(q.cuda() if not q.is_cuda else q, g["k_pages"], g["v_pages"], g["page_table"], g["lens"], context_size, back, sm_scale, True,
                             g.get("k_scale"), g.get("v_scale"), w, **more)
    assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == (B, H)
    o, lse = o.cpu().double(), lse.cpu().double()
    n = max(int(c["lens"].max()), 1) if B else 1
    rel = 2 * dots * (D + 4) * 2**-22 + 2**-20 + n * 2**-23
    step = 0.0 if q.dtype == F32 else torch.finfo(q.dtype).eps / 2
    tol = mass * (rel[..., None] + step) * 1.01 + ref_o.abs() * step * 2 * 1.01 + torch.finfo(q.dtype).tiny * torch.finfo(q.dtype).eps
    assert bool(((o - ref_o).abs() <= tol).all()), float(((o - ref_o).abs() - tol).max())
    empty = ref_w.sum(-1) == 0
    assert (o[empty] == 0).all() and (lse[empty] == 0).all()
    assert bool(((lse - ref_lse).abs() <= (rel + ref_lse.abs() * 2**-22) * 1.5).all())
    if weights is not None:
        got, L = w.cpu().double(), ref_w.shape[-1]
        want = weights.double()
        add = ref_w.view(B, H_kv, group, L)
        want[..., :L] += add.sum(2)
        off = (add * rel.view(B, H_kv, group, 1)).sum(2) * 1.01
        # (a weight below fp32's least normal number, 2^-126, may become 0: nothing bounds it by a part of itself)
        within = (got[..., :L] - want[..., :L]).abs() <= off + (group + 1) * 2**-23 * want[..., :L].abs() + group * 2**-126
        assert bool(within.all())
        untouched = (ref_w.view(B, H_kv, group, L).sum(2) == 0)
        assert torch.equal(w.cpu()[..., :L][untouched], weights[..., :L][untouched]) and torch.equal(w.cpu()[..., L:], weights[..., L:])
    return o, lse


@pytest.mark.parametrize("H,H_kv,D,page,lens,q_dtype,dtype", [
    (4, 4, 64, 16, [37, 1, 0, 64], F32, F32),                       # a length of one, of none, whole pages
    (8, 2, 64, 16, [130, 5], BF16, BF16),
    (8, 2, 128, 64, [700, 64, 65, 63], BF16, BF16),                 # pages that end inside, before and at a tile
    (16, 2, 128, 48, [500, 333], F16, F16),                         # pages that are no power of two
    (32, 1, 128, 32, [257, 90], BF16, BF16),                        # more query heads than a tile has rows
    (24, 8, 64, 1, [70, 3], F16, F16),                              # a row per page
    (20, 1, 64, 128, [1000], F16, F16),
    (12, 4, 128, 8, [90, 800, 7], BF16, BF16),
    (3, 3, 16, 16, [50, 20], BF16, BF16),
    (2, 1, 32, 16, [50, 20], F16, F16),
    (6, 2, 256, 16, [50, 300], F32, F32),
    (5, 5, 256, 32, [100, 0], BF16, BF16),
    (8, 2, 128, 64, [300, 129, 1], BF16, F8),
    (8, 8, 64, 32, [300, 31], F16, F8),
    (6, 1, 128, 16, [77, 256], F32, F8),
    (2, 2, 16, 8, [77], BF16, F8),
    (4, 2, 32, 8, [77], F32, F8),
    (4, 1, 256, 8, [77], F16, F8),
    (16, 16, 64, 32, [513, 512, 511], F16, F16),                    # every head with keys of its own
    (40, 2, 128, 64, [400, 100], BF16, F8),                         # groups of twenty
    (20, 1, 64, 16, [333, 40], BF16, F8),
    (24, 1, 128, 32, [257, 90], F16, F16),
    (17, 1, 64, 16, [257, 90, 0], BF16, BF16),
    (50, 2, 64, 16, [100, 33], F16, F16),                           # more heads than an item takes, unevenly
    (9, 1, 64, 16, [200, 17], F32, F32),
    (24, 2, 128, 48, [200, 17, 1], F32, F32),
    (20, 1, 128, 16, [300], F32, F32),
    (3, 3, 128, 64, [700, 64], F32, F32),
])
@pytest.mark.parametrize("weigh", [False, True])
def test_attention_matches_definition(H, H_kv, D, page, lens, q_dtype, dtype, weigh):
    c = make_cache(len(lens), H_kv, D, page, lens, dtype, stale=float("nan"))
    q = (torch.randn(len(lens), H, D, generator=torch.Generator().manual_seed(7)) * 2).to(q_dtype)
    capacity = c["page_table"].shape[1] * page
    weights = torch.rand(len(lens), H_kv, capacity + 3) if weigh else None
    check_attend(c, q, weights=weights)


@pytest.mark.parametrize("dtype,q_dtype,H,D", [(F32, F32, 2, 64), (BF16, BF16, 8, 128), (F16, F16, 2, 64), (F8, BF16, 4, 128)])
@pytest.mark.parametrize("context_size,back", [(1, 0), (10, 0), (10, 3), (64, 1), (100, 2), (1000, 0), (2**31 - 1, 5), (7, 2**31 - 1)])
def test_attention_with_the_operators_mask(dtype, q_dtype, H, D, context_size, back):
    lens = [1, 10, 11, 64, 65, 640, 500]
    c = make_cache(len(lens), 2, D, 16, lens, dtype, stale=float("inf"))
    q = torch.randn(len(lens), H, D, generator=torch.Generator().manual_seed(8)).to(q_dtype)
    check_attend(c, q, context_size, back, weights=torch.zeros(len(lens), 2, c["page_table"].shape[1] * 16))


@pytest.mark.parametrize("dtype,q_dtype,D", [(F32, F32, 256), (BF16, BF16, 32), (F8, F32, 64), (F16, F16, 16)])
@pytest.mark.parametrize("context_size,back", [(10, 3), (64, 1), (1, 0)])
def test_windows_and_weights_of_the_cuda_core_kernel(dtype, q_dtype, D, context_size, back):
    lens = [1, 64, 65, 0, 640, 500]
    c = make_cache(len(lens), 2, D, 16, lens, dtype, stale=float("nan"), M=60)
    q = torch.randn(len(lens), 6, D, generator=torch.Generator().manual_seed(8)).to(q_dtype)
    check_attend(c, q, context_size, back, weights=torch.rand(len(lens), 2, 60 * 16))


@pytest.mark.parametrize("dtype", [F32, BF16, F8])
def test_attention_splits_long_rows(dtype):
    """One sequence over many blocks, beside short ones that leave most blocks without rows."""
    for lens in ([9001], [3, 20000, 0, 130]):
        c = make_cache(len(lens), 2, 128, 64, lens, dtype)
        q = torch.randn(len(lens), 8, 128, generator=torch.Generator().manual_seed(9)).to(F32 if dtype == F32 else BF16)
        check_attend(c, q, weights=torch.zeros(len(lens), 2, c["page_table"].shape[1] * 64))


@pytest.mark.parametrize("dtype,D,H_kv,B", [(BF16, 128, 8, 260), (F16, 64, 16, 90), (F8, 128, 8, 170), (F32, 64, 8, 260), (F32, 128, 4, 180), (BF16, 32, 8, 90)])
def test_attention_of_many_sequences(dtype, D, H_kv, B):
    """More sequences and heads than there are warps (or blocks) to work on them: several to a warp, some cut in two, one very long, some empty."""
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 90, (B,), generator=g).tolist()
    lens[3], lens[17], lens[B - 1] = 2500, 700, 333
    c = make_cache(B, H_kv, D, 16, lens, dtype)
    q = torch.randn(B, H_kv, D, generator=g).to(F32 if dtype == F32 else F16 if dtype == F16 else BF16)
    check_attend(c, q, weights=torch.zeros(B, H_kv, c["page_table"].shape[1] * 16))


@pytest.mark.parametrize("dtype,D,H_kv,B", [(BF16, 128, 16, 110), (F16, 64, 16, 74), (F8, 64, 16, 73), (F32, 128, 4, 148), (BF16, 256, 8, 70)])
def test_attention_of_sequences_of_one_length(dtype, D, H_kv, B):
    """About as many sequences and heads as there are warps, and much the same lengths: none is cut in two.  Then one that is longer."""
    q = torch.randn(B, H_kv, D, generator=torch.Generator().manual_seed(6)).to(F32 if dtype == F32 else F16 if dtype == F16 else BF16)
    for longest in (70, 300):
        c = make_cache(B, H_kv, D, 16, [60 + b % 11 for b in range(B - 1)] + [longest], dtype, M=20)
        check_attend(c, q, weights=torch.zeros(B, H_kv, 320))


@pytest.mark.parametrize("dtype", [F32, F16, F8])
def test_attention_masks_rows_without_a_page(dtype):
    c = make_cache(4, 2, 64, 16, [100, 100, 90, 33], dtype, stale=float("nan"))
    P = c["k_pages"].shape[0]
    c["page_table"][0, 2], c["page_table"][0, 6], c["page_table"][1] = -1, P, -7
    c["page_table"][2, 0], c["page_table"][3, 2] = 2**31 - 1, -2**31
    q = torch.randn(4, 4, 64).to(F32 if dtype == F32 else F16)
    check_attend(c, q, weights=torch.zeros(4, 2, c["page_table"].shape[1] * 16))
    check_attend(c, q, 16, 1)

def test_a_windows_weights_need_no_workspace_of_the_tables_width():
    """Room for scores follows the rows that a token can see: a table for a long context costs a windowed step nothing."""
    from kernels_b200.streaming_attention import paged_attention

    lens, M = [1000, 64, 129, 0, 700], 65536
    c = make_cache(5, 2, 64, 16, lens, BF16)
    wide = torch.full((5, M), -1, dtype=torch.int32)
    wide[:, : c["page_table"].shape[1]] = c["page_table"]
    q = torch.randn(5, 8, 64).bfloat16()
    for context_size, back in ((128, 1), (1, 0), (64, 3)):
        weights = torch.rand(5, 2, 1008)
        check_attend(c, q, context_size, back, weights=weights)
        g = cuda(c)
        tight, broad = (torch.zeros(5, 2, n, device="cuda") for n in (1008, M * 16))
        args = (q.cuda(), g["k_pages"], g["v_pages"])
        a = paged_attention(*args, g["page_table"], g["lens"], context_size, back, weights=tight)
        table = wide.cuda()
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        b = paged_attention(*args, table, g["lens"], context_size, back, weights=broad)
        assert torch.cuda.max_memory_allocated() - before < 32 << 20  # (scores for the table's width: 160 MB)
        assert torch.equal(a, b) and torch.equal(tight, broad[..., :1008]) and not broad[..., 1008:].any()


def test_attention_lengths_beyond_the_table_are_clamped():
    c = make_cache(3, 2, 64, 16, [64, 64, 64], F16)
    c["lens"][:] = torch.tensor([65, 2**31 - 1, -3])
    check_attend(c, torch.randn(3, 4, 64).half(), weights=torch.zeros(3, 2, 64))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_extreme_scores(dtype):
    """Scores far apart and far from zero: rows one after the other raise the maximum, or leave every later one at 0."""
    c = make_cache(2, 1, 64, 16, [300, 300], dtype)
    ramp = torch.linspace(-3, 3, 300)
    for r in range(300):
        for b, x in enumerate((ramp[r], ramp[299 - r])):
            c["k_pages"][c["page_table"][b, r // 16], 0, r % 16] = float(x)
    q = torch.full((2, 2, 64), 4.0, dtype=dtype)
    check_attend(c, q, weights=torch.zeros(2, 1, c["page_table"].shape[1] * 16))
    check_attend(c, q, sm_scale=-1.0)
    check_attend(c, q, sm_scale=0.0)


def test_attention_nan_and_infinite_rows_stay_in_their_heads():
    from kernels_b200.streaming_attention import paged_attention

    for dtype in (F32, BF16):
        c = make_cache(2, 2, 128, 16, [200, 200], dtype)
        at = c["page_table"][0, 3]
        c["v_pages"][at, 0, 5, 7] = float("nan")
        c["k_pages"][c["page_table"][1, 2], 1, 0] = float("nan")
        q = torch.randn(2, 4, 128).to(dtype)
        g = cuda(c)
        o, lse = paged_attention(q.cuda(), g["k_pages"], g["v_pages"], g["page_table"], g["lens"], return_lse=True)
        assert o[0, :2, 7].isnan().all() and not o[0, :, :7].isnan().any() and not o[0, 2:].isnan().any() and not lse[0].isnan().any()
        assert o[1, 2:].isnan().all() and lse[1, 2:].isnan().all() and not o[1, :2].isnan().any()


@pytest.mark.parametrize("H,D,q_dtype", [(4, 64, BF16), (8, 128, F16), (20, 64, F16), (40, 128, BF16), (4, 32, BF16), (4, 64, F32)])
@pytest.mark.parametrize("n", [1, 90, 9001])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_attention_over_8_bit_pages_with_an_infinite_value(H, D, q_dtype, n, bad):
    """A value row with an infinity is written with an infinite scale: the heads that see it are NaN, cut into parts or not (0 times infinity), but
    their log-sum-exp and their rows' weights, which do not depend on the values, are those of the definition."""
    from kernels_b200.streaming_attention import paged_attention, paged_cache_write

    lens = [n, 33]
    c = make_cache(2, 2, D, 16, lens, F8)
    g = cuda(c)
    v = torch.randn(2, 2, 1, D)
    v[0, 1, 0, 3] = bad
    k = torch.randn(2, 2, 1, D)
    paged_cache_write(k.cuda(), v.cuda(), g["k_pages"], g["v_pages"], g["page_table"], g["lens"], k_scale=g["k_scale"], v_scale=g["v_scale"])
    scale = g["v_scale"].cpu()
    assert int((~scale.isfinite()).sum()) == 1
    c = {name: x.cpu() for name, x in g.items()}
    q = torch.randn(2, H, D, generator=torch.Generator().manual_seed(7)).to(q_dtype)
    L = c["page_table"].shape[1] * 16
    ref_o, ref_lse, ref_w, (dots, _) = PO.attend(q, c["k_pages"], c["v_pages"], c["page_table"], c["lens"], k_scale=c["k_scale"], v_scale=c["v_scale"])
    assert ref_o[0, H // 2:].isnan().all() and not ref_o[0, : H // 2].isnan().any() and not ref_o[1].isnan().any()
    w = torch.zeros(2, 2, L, device="cuda")
    o, lse = paged_attention(q.cuda(), *(g[name] for name in ("k_pages", "v_pages", "page_table", "lens")), return_lse=True,
                             k_scale=g["k_scale"], v_scale=g["v_scale"], weights=w)
    assert torch.equal(o.cpu().isnan(), ref_o.isnan())
    rel = 2 * dots * (D + 4) * 2**-22 + 2**-20 + n * 2**-23  # as above
    assert bool(((lse.cpu().double() - ref_lse).abs() <= (rel + ref_lse.abs() * 2**-22) * 1.5).all())
    add = ref_w.view(2, 2, H // 2, L)
    off = (add * rel.view(2, 2, H // 2, 1)).sum(2) * 1.01 + (H // 2 + 1) * 2**-23 * add.sum(2) + H // 2 * 2**-126
    assert bool(((w.cpu().double() - add.sum(2)).abs() <= off).all())


def test_attention_over_very_many_rows_of_scale_zero():
    """Value scales of 0 leave the rows' weights as they are: their sum stays within fp32 however many there are.  (One sequence's pages read by 64
    sequences, so that a stretch of the line is about fourteen thousand rows; the first rows' scores lie 7.9 below the others', just too little to raise the maximum.)"""
    from kernels_b200.streaming_attention import paged_attention

    B, H_kv, D, page, n = 64, 8, 64, 64, 32768
    c = make_cache(1, H_kv, D, page, [n], F8)
    c["k_pages"] = torch.zeros(c["k_pages"].shape).to(F8)
    c["k_scale"].fill_(1.0)
    c["v_scale"].zero_()
    rows = torch.zeros(n)
    rows[32:] = 1.0
    k = c["k_pages"].float()
    for m in range(n // page):
        k[c["page_table"][0, m], :, :, 0] = rows[m * page: (m + 1) * page]
    c["k_pages"] = k.to(F8)
    g = cuda(c)
    q = torch.zeros(B, H_kv, D, dtype=F16, device="cuda")
    q[..., 0] = 1.0
    step = 7.875  # base-2 steps between the two scores
    o, lse = paged_attention(q, g["k_pages"], g["v_pages"], g["page_table"].expand(B, -1), g["lens"].expand(B), sm_scale=step / 1.4426950408889634, return_lse=True,
                             k_scale=g["k_scale"], v_scale=g["v_scale"])
    want = torch.log2(torch.tensor((n - 32) * 2.0**step + 32, dtype=torch.float64))
    assert (o == 0).all()
    # a weight is off by 2^-20 of itself (its argument, up to 2^7, is rounded to 2^-18 and less where it counts), a sum of n terms by n 2^-24
    assert ((lse.cpu().double() - want).abs() <= (2**-17 + n * 2**-24) * 1.5).all()


@pytest.mark.parametrize("D,H,q_dtype", [(64, 4, BF16), (128, 8, F16), (128, 40, BF16), (32, 4, BF16)])
@pytest.mark.parametrize("low,high", [(-40, 40), (-75, 10), (0, 85), (-100, -90), (60, 62)])
def test_attention_over_8_bit_pages_of_any_scales(D, H, q_dtype, low, high):
    """Value scales spread over many powers of two within a sequence, some of them 0 or negative.

    Weights are multiplied as f16 numbers p v_scale whose largest is 2^7 at least: what lies below f16's least step, 2^-24, is off by half of it,
    2^-32 of the largest p |v_scale|, times an element of 448 at most.  Where all scales are below 2^-80 the largest is that much smaller, and so
    are the outputs: 2^-80 in its place.  A weight's argument is at most 2^8 in magnitude: rounded by 2^-17, so the weight by 2^-17 of itself."""
    from kernels_b200.streaming_attention import paged_attention

    gen = torch.Generator().manual_seed(D + H)
    lens = [700, 41, 1]
    c = make_cache(3, 2, D, 16, lens, F8)
    spread = torch.rand(c["v_scale"].shape, generator=gen) * (high - low) + low
    c["v_scale"] = torch.exp2(spread) * torch.where(torch.rand(spread.shape, generator=gen) < 0.2, -1.0, 1.0)
    c["v_scale"][torch.rand(spread.shape, generator=gen) < 0.05] = 0.0
    q = torch.randn(3, H, D, generator=gen).to(q_dtype)
    ref_o, ref_lse, ref_w, (dots, mass) = PO.attend(q, c["k_pages"], c["v_pages"], c["page_table"], c["lens"], k_scale=c["k_scale"], v_scale=c["v_scale"])
    g = cuda(c)
    L = c["page_table"].shape[1] * 16
    w = torch.zeros(3, 2, L, device="cuda")
    o, lse = paged_attention(q.cuda(), *(g[n] for n in ("k_pages", "v_pages", "page_table", "lens")), return_lse=True, k_scale=g["k_scale"],
                             v_scale=g["v_scale"], weights=w)
    o, lse = o.cpu().double(), lse.cpu().double()
    group = H // 2
    row_scale = torch.zeros(3, 2, L, dtype=torch.float64)
    for b, n in enumerate(lens):
        for r in range(n):
            row_scale[b, :, r] = c["v_scale"][c["page_table"][b, r // 16], :, r % 16].double()
    top = (ref_w.view(3, 2, group, L) * row_scale[:, :, None].abs().clamp_min(2.0**-80)).amax(-1).view(3, H)
    rel = 2 * dots * (D + 4) * 2**-22 + 2**-16 + max(lens) * 2**-23
    step = torch.finfo(q_dtype).eps / 2
    least = torch.finfo(q_dtype).tiny * torch.finfo(q_dtype).eps
    weight_step = 2.0**-11  # f16 weights
    tol = mass * (rel[..., None] + weight_step) * 1.01 + ref_o.abs() * step * 1.01 + least + (top * max(lens) * 2.0**-32 * 448)[..., None]
    fits = ref_o.abs() + tol < torch.finfo(q_dtype).max  # (what leaves fp16 is infinite)
    assert bool(((o - ref_o).abs() <= tol)[fits].all()) and not o.isnan().any()
    assert bool(((lse - ref_lse).abs() <= (rel + (ref_lse.abs() + 100) * 2**-22) * 1.5).all())
    add = ref_w.view(3, 2, group, L)
    off = (add * rel.view(3, 2, group, 1)).sum(2) * 1.5 + (group + 1) * 2**-23 * add.sum(2) + group * 2**-126
    assert bool(((w.cpu().double() - add.sum(2)).abs() <= off).all())


@pytest.mark.parametrize("size", [1e-36, 1e-30, 1e-20, 1e20, 1e30, 1e36])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_over_8_bit_pages_of_far_queries(size, D):
    """bf16 queries far from 1, with a scale that brings their scores back."""
    c = make_cache(2, 2, D, 16, [300, 45], F8)
    q = (torch.randn(2, 4, D, generator=torch.Generator().manual_seed(3)) * size).to(BF16)
    check_attend(c, q, sm_scale=0.125 / size, weights=torch.zeros(2, 2, c["page_table"].shape[1] * 16))


@pytest.mark.parametrize("q_dtype", [F16, BF16, F32])
def test_attention_extreme_scores_over_8_bit_pages(q_dtype):
    """Rows one after the other that raise the maximum by a little or a lot, and the other way round."""
    c = make_cache(2, 1, 64, 16, [300, 300], F8)
    k, ramp = c["k_pages"].float(), torch.linspace(-3, 3, 300)
    for r in range(300):
        for b, x in enumerate((ramp[r], ramp[299 - r])):
            k[c["page_table"][b, r // 16], 0, r % 16] = float(x)
    c["k_pages"] = k.to(F8)
    c["k_scale"].fill_(1.0)
    q = torch.full((2, 2, 64), 4.0, dtype=q_dtype)
    for scale in (None, -1.0, 0.0, 0.02):
        check_attend(c, q, sm_scale=scale, weights=torch.zeros(2, 1, c["page_table"].shape[1] * 16))


@pytest.mark.parametrize("dtype", [F32, F16, F8])
def test_attention_takes_any_layout(dtype):
    """A [P, page, H_kv, D] pool, pages apart, rows off the 16-byte boundaries; tables and lengths as views; q in another order."""
    from kernels_b200.streaming_attention import paged_attention

    c = make_cache(3, 2, 64, 16, [100, 7, 61], dtype)
    q = torch.randn(3, 4, 64).to(F32 if dtype == F32 else F16)
    scale = {n: c.get(n) for n in ("k_scale", "v_scale")}
    ref, _ = check_attend(c, q)
    g = cuda(c)

    def other(x):  # heads inside rows
        return x.transpose(1, 2).contiguous().transpose(1, 2)

    def apart(x):
        y = torch.zeros(*x.shape[:-1], x.shape[-1] + 5, dtype=torch.uint8 if dtype == F8 else dtype, device="cuda")
        y = y.view(dtype)[..., 3: 3 + x.shape[-1]] if dtype != F8 else y[..., 3: 3 + x.shape[-1]]
        (y if dtype != F8 else y).copy_(x if dtype != F8 else x.view(torch.uint8))
        return y.view(F8) if dtype == F8 else y

    table = torch.zeros(3, 2 * g["page_table"].shape[1], dtype=torch.int32, device="cuda")[:, ::2]
    table.copy_(g["page_table"])
    lens = torch.zeros(6, dtype=torch.int32, device="cuda")[::2]
    lens.copy_(g["lens"])
    for form in (other, apart):
        changed = dict(g, k_pages=form(g["k_pages"]), v_pages=form(g["v_pages"]), page_table=table, lens=lens)
        if dtype == F8:
            changed |= dict(k_scale=other(g["k_scale"]), v_scale=g["v_scale"].transpose(0, 2).contiguous().transpose(0, 2))
        check_attend(c, q, on_gpu=changed)
    check_attend(c, q, on_gpu=dict(g, v_pages=other(g["v_pages"])))  # keys and values of different layouts
    del scale, ref
    for qs in (q.cuda().transpose(0, 1).contiguous().transpose(0, 1), q.cuda().transpose(1, 2).contiguous().transpose(1, 2)):
        a = paged_attention(qs, g["k_pages"], g["v_pages"], g["page_table"], g["lens"], k_scale=g.get("k_scale"), v_scale=g.get("v_scale"))
        b = paged_attention(q.cuda(), g["k_pages"], g["v_pages"], g["page_table"], g["lens"], k_scale=g.get("k_scale"), v_scale=g.get("v_scale"))
        assert torch.equal(a, b)


def test_a_cache_past_32_bit_offsets():
    """The last pages of pools of 2^32 elements and more: attended with, written, evicted from."""
    from kernels_b200.streaming_attention import paged_cache_evict, paged_cache_write

    P, page, D = 17000, 2048, 128
    k, v = (torch.zeros(P, 1, page, D, dtype=F16, device="cuda") for _ in range(2))
    assert k.numel() > 2**32
    c = make_cache(1, 1, D, page, [3000], F16, spare=0)
    order = c["page_table"][0].long()
    table = torch.tensor([[P - 1, P - 2]], dtype=torch.int32)
    for pool, small in ((k, c["k_pages"]), (v, c["v_pages"])):
        pool[P - 1], pool[P - 2] = small[order[0]].cuda(), small[order[1]].cuda()
    q = torch.randn(1, 2, D).half()
    g = dict(k_pages=k, v_pages=v, page_table=table.cuda(), lens=c["lens"].cuda())
    check_attend(c, q, on_gpu=g)
    check_attend(c, q, on_gpu=dict(g, v_pages=v.view(P, page, 1, D).transpose(1, 2)))  # (another layout on paper: the generic kernel)
    weights, positions = make_books(1, 1, 2 * page)
    books = weights.cuda(), positions.cuda()
    x, y = (torch.randn(1, 1, 5, D).half() for _ in range(2))
    c["lens"] += 5
    g["lens"] += 5
    PO.write(x, y, c["k_pages"], c["v_pages"], c["page_table"], c["lens"], None, None, weights, positions)
    paged_cache_write(x.cuda(), y.cuda(), *g.values(), weights=books[0], row_positions=books[1])
    PO.evict(c["k_pages"], c["v_pages"], c["page_table"], c["lens"], weights, positions, 2500, 100)
    paged_cache_evict(*g.values(), *books, 2500, 100)
    for pool, small in ((k, c["k_pages"]), (v, c["v_pages"])):
        assert torch.equal(pool[P - 1].cpu(), small[order[0]]) and torch.equal(pool[P - 2].cpu(), small[order[1]]) and not pool[: P - 2].any()
    assert torch.equal(books[0].cpu(), weights) and torch.equal(books[1].cpu(), positions) and g["lens"].tolist() == [2500]


def test_attention_same_inputs_same_bits():
    from kernels_b200.streaming_attention import paged_attention

    g = cuda(make_cache(3, 2, 128, 64, [5000, 100, 2100], BF16))
    q = torch.randn(3, 16, 128).bfloat16().cuda()
    runs = []
    for _ in range(3):
        w = torch.zeros(3, 2, g["page_table"].shape[1] * 64, device="cuda")
        runs.append((*paged_attention(q, g["k_pages"], g["v_pages"], g["page_table"], g["lens"], return_lse=True, weights=w), w))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_attention_empty_calls():
    from kernels_b200.streaming_attention import paged_attention

    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    pages = torch.zeros(4, 2, 16, 64, dtype=F16, device="cuda")
    assert paged_attention(pages[:0, 0, :4], pages, pages, i(0, 3), i(0)).shape == (0, 4, 64)
    q = torch.ones(3, 4, 64, dtype=F16, device="cuda")
    for args in ((pages, pages, i(3, 0), i(3) + 5), (pages[:0], pages[:0], i(3, 2), i(3) + 20), (pages, pages, i(3, 2), i(3))):
        o, lse = paged_attention(q, *args, return_lse=True)
        assert (o == 0).all() and (lse == 0).all()


# ---- write ---------------------------------------------------------------------------------------------------------


def check_write(c, k, v, new_lens=None, positions=None, book=True, kg=None, vg=None):
    from kernels_b200.streaming_attention import paged_cache_write

    H_kv, L = k.shape[1], c["page_table"].shape[1] * c["k_pages"].shape[2]
    ref = {n: x.clone() for n, x in c.items()}
    more = dict(weights=torch.rand(len(c["lens"]), H_kv, L + 2), row_positions=torch.randint(0, 99, (len(c["lens"]), H_kv, L), dtype=torch.int32)) if book else {}
    g = cuda(c | more)
    PO.write(k, v, ref["k_pages"], ref["v_pages"], ref["page_table"], ref["lens"], new_lens, positions, more.get("weights"), more.get("row_positions"),
             ref.get("k_scale"), ref.get("v_scale"))
    paged_cache_write(k.cuda() if kg is None else kg, v.cuda() if vg is None else vg, g["k_pages"], g["v_pages"], g["page_table"], g["lens"],
                      None if new_lens is None else new_lens.cuda(), None if positions is None else positions.cuda(), g.get("weights"),
                      g.get("row_positions"), g.get("k_scale"), g.get("v_scale"))
    for n, x in (ref | more).items():
        y = g[n].cpu()
        x, y = (t.view(torch.uint8) if t.dtype == F8 else t for t in (x, y))
        assert torch.equal(x, y) if not x.is_floating_point() else torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0)), n
    return g


@pytest.mark.parametrize("H_kv,D,page,lens,T,new,dtype,cache", [
    (2, 64, 16, [1, 16, 17, 40], 1, None, F16, F16),                     # the newest token of every sequence
    (8, 128, 64, [300, 64, 500], 64, None, BF16, BF16),
    (3, 128, 48, [100, 60, 7], 60, [60, 10, 7], BF16, F8),               # ragged prompts
    (2, 64, 8, [33, 5, 0, 2], 9, [9, 0, 4, 9], F32, F32),                # nothing new; more new tokens than rows
    (1, 16, 16, [20], 20, None, F16, F8),
    (2, 32, 16, [20, 3], 3, None, F32, F8),
    (2, 256, 16, [20, 3], 3, [2, 3], F32, F8),
    (2, 256, 16, [20, 3], 3, [2, 3], F32, F32),
    (5, 16, 4, [9], 9, [-1], BF16, BF16),
])
@pytest.mark.parametrize("positions", [False, True])
def test_write_matches_definition(H_kv, D, page, lens, T, new, dtype, cache, positions):
    B = len(lens)
    c = make_cache(B, H_kv, D, page, lens, cache)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(B, H_kv, T, D, generator=g).to(dtype) for _ in range(2))
    k[0, 0, 0] = 0  # a row of zeros has the least scale
    new = None if new is None else torch.tensor(new, dtype=torch.int32)
    check_write(c, k, v, new, torch.randint(0, 10**6, (B, T), dtype=torch.int32) if positions else None)
    check_write(c, k, v, new, book=False)


@pytest.mark.parametrize("cache", [F16, F8])
def test_write_drops_rows_without_a_page_or_outside_the_table(cache):
    c = make_cache(4, 2, 64, 16, [80, 80, 80, 80], cache)
    c["page_table"][0, 1], c["page_table"][1] = -1, c["k_pages"].shape[0]
    c["lens"] = torch.tensor([80, 80, 100, 2**31 - 1], dtype=torch.int32)
    k, v = (torch.randn(4, 2, 70, 64).half() for _ in range(2))
    check_write(c, k, v)
    c["lens"] = torch.tensor([-5, -2**31, 3, 69], dtype=torch.int32)
    check_write(c, k, v)


def test_write_special_values_and_layouts():
    c = make_cache(2, 2, 64, 16, [30, 30], F8)
    k, v = (torch.randn(2, 2, 20, 64).bfloat16() for _ in range(2))
    k[0, 0, 3, 5], v[1, 1, 2, 1], k[1, 0, 0] = float("nan"), float("inf"), 1e-30
    g = check_write_special(c, k, v)
    assert g["k_scale"].isnan().sum() == 1 and g["v_scale"].isinf().sum() == 1
    for cache in (F8, BF16):
        c = make_cache(2, 2, 64, 16, [30, 30], cache)
        k, v = (torch.randn(2, 2, 20, 64).bfloat16() for _ in range(2))
        kt = k.transpose(1, 2).contiguous().cuda().transpose(1, 2)
        vo = torch.zeros(2, 2, 20, 67, dtype=BF16, device="cuda")[..., 3:]
        vo.copy_(v)
        check_write(c, k, v, kg=kt, vg=vo)
        check_write(c, k, v, kg=k.cuda().transpose(2, 3).contiguous().transpose(2, 3))


def check_write_special(c, k, v):
    from kernels_b200.streaming_attention import paged_cache_write

    g = cuda(c)
    paged_cache_write(k.cuda(), v.cuda(), g["k_pages"], g["v_pages"], g["page_table"], g["lens"], k_scale=g["k_scale"], v_scale=g["v_scale"])
    ref = {n: x.clone() for n, x in c.items()}
    plain = torch.ones(2, 2, 20, dtype=torch.bool)
    PO.write(k, v, ref["k_pages"], ref["v_pages"], ref["page_table"], ref["lens"], None, None, None, None, ref["k_scale"], ref["v_scale"])
    for b in range(2):
        for h in range(2):
            for t in range(20):
                at = PO.place(c["page_table"][b], 10 + t, 16, c["k_pages"].shape[0])
                for n, x in (("k", k), ("v", v)):
                    if x[b, h, t].isfinite().all():
                        assert torch.equal(g[n + "_pages"].cpu().view(torch.uint8)[at[0], h, at[1]], ref[n + "_pages"].view(torch.uint8)[at[0], h, at[1]])
    del plain
    return g


# ---- evict ---------------------------------------------------------------------------------------------------------


def make_books(B, H_kv, L, seed=0, ties=False):
    g = torch.Generator().manual_seed(seed)
    w = torch.rand(B, H_kv, L, generator=g) ** 3
    if ties:
        w = (w * 4).round() / 4
    pos = torch.rand(B, H_kv, L, generator=g).argsort(-1).to(torch.int32) + 1000
    return w, pos


def check_evict(c, w, pos, budget, recent, in_place=True):
    from kernels_b200.streaming_attention import paged_cache_evict

    ref = {n: x.clone() for n, x in (c | dict(weights=w, row_positions=pos)).items()}
    g = cuda(ref)
    PO.evict(ref["k_pages"], ref["v_pages"], ref["page_table"], ref["lens"], ref["weights"], ref["row_positions"], budget, recent, ref.get("k_scale"),
             ref.get("v_scale"))
    args = (g["k_pages"], g["v_pages"], g["page_table"], g["lens"], g["weights"], g["row_positions"], budget, recent, g.get("k_scale"), g.get("v_scale"))
    if in_place:
        got = paged_cache_evict(*args)
        assert got[0] is g["lens"] and got[1] is g["weights"] and got[2] is g["row_positions"]
    else:
        out = (torch.full_like(g["lens"], -9), torch.full_like(g["weights"], -9.0), torch.full_like(g["row_positions"], -9))
        before = [g[n].clone() for n in ("lens", "weights", "row_positions")]
        got = paged_cache_evict(*args, out=out)
        assert all(torch.equal(x, g[n]) for x, n in zip(before, ("lens", "weights", "row_positions")))
        lens = ref["lens"].clamp(0, c["page_table"].shape[1] * c["k_pages"].shape[2])
        stays = torch.arange(w.shape[-1])[None, None] < lens[:, None, None]
        ref["weights"], ref["row_positions"] = torch.where(stays, ref["weights"], -9.0), torch.where(stays, ref["row_positions"], -9)
        g |= dict(zip(("lens", "weights", "row_positions"), got))
    for n, x in ref.items():
        y = g[n].cpu()
        x, y = (t.view(torch.uint8) if t.dtype == F8 else t for t in (x, y))
        if x.is_floating_point():
            x, y = x.nan_to_num(-3.0), y.nan_to_num(-3.0)
        assert torch.equal(x, y), n
    return g


@pytest.mark.parametrize("H_kv,D,page,lens,dtype,budget,recent", [
    (2, 64, 16, [65, 64, 63, 0], F16, 64, 8),               # one row over, exactly full, not full, empty
    (3, 128, 16, [500, 300, 100], BF16, 100, 20),
    (2, 64, 48, [1500, 2049], F32, 700, 0),
    (1, 16, 8, [40], BF16, 1, 0),                           # a single row stays
    (2, 128, 64, [900, 1025], F8, 333, 333),                # nothing but the newest
    (2, 64, 16, [400], F16, 100, 1000),                     # more newest rows than the budget
    (2, 64, 1, [33, 70], F16, 32, 5),
    (2, 32, 16, [200, 90], F8, 128, 16),
    (1, 256, 16, [200, 90], F32, 64, 16),
    (2, 64, 16, [50, 60], F16, 10**9, 4),
    (1, 64, 64, [40000, 16385, 30], F16, 5000, 100),        # longer than a block holds, shorter than its cluster
    (1, 16, 64, [140000, 100], F16, 70000, 0),              # longer than a cluster holds
    (2, 16, 64, [20000, 8000], F16, 8100, 16),              # half of a cluster without rows
])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_matches_definition(H_kv, D, page, lens, dtype, budget, recent, ties):
    c = make_cache(len(lens), H_kv, D, page, lens, dtype)
    w, pos = make_books(len(lens), H_kv, c["page_table"].shape[1] * page, ties=ties)
    check_evict(c, w, pos, budget, recent)
    check_evict(c, w, pos, budget, recent, in_place=False)

@pytest.mark.parametrize("H_kv,page,lens,budget,recent", [
    (2, 16, [65], 64, 100),                    # one row over, every one of them recent
    (2, 16, [400, 70, 64], 64, 65),
    (1, 64, [40000, 20000], 5000, 2**31 - 1),  # a cluster
    (1, 64, [140000], 70000, 100000),          # longer than a cluster holds
    (2, 16, [3000], 1000, 2000),               # more recent rows than the budget, and others besides
])
@pytest.mark.parametrize("shuffled", [False, True])
def test_evict_keeps_the_newest_of_more_recent_rows_than_the_budget(H_kv, page, lens, budget, recent, shuffled):
    """Weights say nothing where the recent rows alone pass the budget: the newest of them stay, so that a token just written is never the one that goes."""
    c = make_cache(len(lens), H_kv, 16, page, lens, F16)
    L = c["page_table"].shape[1] * page
    w, pos = make_books(len(lens), H_kv, L)
    if not shuffled:
        pos = torch.arange(L, dtype=torch.int32).expand(len(lens), H_kv, L).contiguous()
    g = check_evict(c, w, pos, budget, recent)
    check_evict(c, w, pos, budget, recent, in_place=False)
    for b, n in enumerate(lens):
        for h in range(H_kv):
            kept, rows = set(g["row_positions"][b, h, : min(n, budget)].tolist()), pos[b, h, :n]
            newest = rows[rows > int(rows.max()) - recent].sort(descending=True).values[:budget]
            assert set(newest.tolist()) <= kept and (n <= budget or len(newest) < budget or set(newest.tolist()) == kept)


def test_a_cache_whose_budget_is_smaller_than_its_window_goes_on():
    """Token after token, the cache holds the newest ``budget`` of them."""
    from kernels_b200.streaming_attention import paged_cache_evict, paged_cache_write

    c = make_cache(1, 2, 64, 16, [96], F16)
    g = cuda(c)
    g["lens"].zero_()
    w, pos = torch.zeros(1, 2, 96, device="cuda"), torch.zeros(1, 2, 96, dtype=torch.int32, device="cuda")
    pages = tuple(g[n] for n in ("k_pages", "v_pages", "page_table", "lens"))
    for t in range(150):
        g["lens"] += 1
        x = torch.full((1, 2, 1, 64), float(t), dtype=F16, device="cuda")
        paged_cache_write(x, x, *pages, positions=torch.tensor([[t]], dtype=torch.int32, device="cuda"), weights=w, row_positions=pos)
        w[:, :, 0] = 100.0  # (the oldest place is the heaviest)
        paged_cache_evict(*pages, w, pos, 64, 100)
    assert g["lens"].tolist() == [64]
    for h in range(2):
        assert sorted(pos[0, h, :64].tolist()) == list(range(86, 150))
        rows = [g["k_pages"][g["page_table"][0, r // 16], h, r % 16, 0].item() for r in range(64)]
        assert rows == pos[0, h, :64].tolist()


def test_evict_special_weights_and_positions():
    c = make_cache(3, 2, 64, 16, [100, 100, 100], F16)
    w, pos = make_books(3, 2, c["page_table"].shape[1] * 16)
    w[0, 0, ::3], w[0, 1, ::7], w[1, 0], w[1, 1, ::2] = float("nan"), float("inf"), 0.0, -1.0
    w[2, 0, ::2], w[2, 0, 1::2], w[2, 1] = -0.0, 0.0, -float("inf")
    pos[0, 0], pos[1, 1, 40:], pos[2, 1, :3] = 5, 2**31 - 1, -2**31
    for budget, recent in ((50, 10), (33, 0), (99, 99), (20, 2**31 - 1)):
        check_evict(c, w, pos, budget, recent)  # (the definition compares numbers: both zeros are one)


def test_evict_leaves_rows_without_a_page_alone():
    c = make_cache(3, 2, 64, 16, [100, 100, 100], F16)
    P = c["k_pages"].shape[0]
    c["page_table"][0, 1], c["page_table"][0, 5], c["page_table"][1], c["page_table"][2, 6] = -1, P, -2**31, 2**31 - 1
    c["lens"] = torch.tensor([100, 100, 2**31 - 1], dtype=torch.int32)
    w, pos = make_books(3, 2, c["page_table"].shape[1] * 16 + 8)
    check_evict(c, w, pos, 50, 5)
    check_evict(c, w, pos, 50, 5, in_place=False)
    c["lens"] = torch.tensor([-1, 100, -2**31], dtype=torch.int32)
    check_evict(c, w, pos, 60, 5)

@pytest.mark.parametrize("page,n,budget,recent,gone", [
    (16, 100, 50, 5, [1, 5]), (16, 100, 50, 5, [6]), (16, 100, 50, 0, [0, 1, 2]), (16, 100, 50, 5, [0, 1, 2, 3]), (16, 100, 50, 200, [0, 4]), (1, 60, 30, 3, [0, 3, 7, 29, 30, 31, 59]),
    (16, 100, 50, 5, [3, 4, 5, 6]), (64, 40000, 5000, 100, [0, 9, 78, 79, 300, 624]), (64, 140000, 70000, 0, [3, 1093, 1094, 2000]),
])
def test_evict_passes_over_rows_without_a_page(page, n, budget, recent, gone):
    """A row without a page holds nothing: it is not kept in a place that others could fill, and no kept row moves into a place without one.  Every visible
    row that is left has its own keys and values beside its own weight and position."""
    c = make_cache(2, 2, 16, page, [n, n], F32)
    c["page_table"][0, gone] = torch.tensor([-1, c["k_pages"].shape[0], 2**31 - 1, -2**31])[torch.arange(len(gone)) % 4].to(torch.int32)
    L = c["page_table"].shape[1] * page
    w, pos = make_books(2, 2, L)
    for h in range(2):  # rows are told by their positions (below 2^24)
        for b in range(2):
            for name in ("k_pages", "v_pages"):
                at = c["page_table"][b].long()
                held = (at >= 0) & (at < c["k_pages"].shape[0])
                c[name][at[held], h] = pos[b, h].view(-1, page)[held][..., None].expand(-1, -1, 16).float()
    g = check_evict(c, w, pos, budget, recent)
    check_evict(c, w, pos, budget, recent, in_place=False)
    held = torch.tensor([PO.place(c["page_table"][0], r, page, c["k_pages"].shape[0]) is not None for r in range(n)])
    for h in range(2):
        seen = held[:budget].nonzero()[:, 0]
        at = c["page_table"][0].long()[seen // page]
        for name in ("k_pages", "v_pages"):
            rows = g[name].cpu()[at, h, seen % page]
            assert torch.equal(rows, g["row_positions"].cpu()[0, h, seen][:, None].expand(-1, 16).float())
        left = set(g["row_positions"][0, h, seen.cuda()].tolist())
        assert len(left) == len(seen) and left <= set(pos[0, h, :n][held].tolist())


def test_evict_from_strided_tables_and_from_no_pages_at_all():
    c = make_cache(2, 2, 64, 16, [100, 90], F16)
    w, pos = make_books(2, 2, c["page_table"].shape[1] * 16)
    from kernels_b200.streaming_attention import paged_cache_evict

    for gone in ([], [1, 5]):
        c["page_table"][0, gone] = -1
        want, g = check_evict(c, w, pos, 50, 5), cuda(c | dict(weights=w, row_positions=pos))
        wide = torch.full((2, 3 * c["page_table"].shape[1]), 10**6, dtype=torch.int32, device="cuda")[:, ::3]
        wide.copy_(g["page_table"])
        paged_cache_evict(g["k_pages"], g["v_pages"], wide, g["lens"], g["weights"], g["row_positions"], 50, 5)
        assert all(torch.equal(want[n], g[n]) for n in g)
    none = dict(c, k_pages=c["k_pages"][:0], v_pages=c["v_pages"][:0])
    g = check_evict(none, w, pos, 50, 5)
    assert g["lens"].tolist() == [50, 50] and torch.equal(g["weights"].cpu(), w) and torch.equal(g["row_positions"].cpu(), pos)


def test_evict_layouts():
    c = make_cache(2, 2, 64, 16, [200, 150], F16)
    w, pos = make_books(2, 2, c["page_table"].shape[1] * 16)
    from kernels_b200.streaming_attention import paged_cache_evict

    ref = check_evict(c, w, pos, 64, 8)
    g = cuda(c)
    k, v = g["k_pages"].transpose(1, 2).contiguous().transpose(1, 2), torch.zeros(*g["v_pages"].shape[:3], 67, dtype=F16, device="cuda")[..., 3:]
    v.copy_(g["v_pages"])
    wt, pt = w.cuda().transpose(0, 1).contiguous().transpose(0, 1), torch.zeros(2, 2, w.shape[2] + 5, dtype=torch.int32, device="cuda")[..., :w.shape[2]]
    pt.copy_(pos)
    lens = torch.zeros(4, dtype=torch.int32, device="cuda")[::2]
    lens.copy_(g["lens"])
    paged_cache_evict(k, v, g["page_table"], lens, wt, pt, 64, 8)
    for x, n in ((k, "k_pages"), (v, "v_pages"), (lens, "lens"), (wt, "weights"), (pt, "row_positions")):
        assert torch.equal(x, ref[n]), n


# ---- together ------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F8), (F32, F32)])
def test_decoding_with_a_budget_matches_the_definitions(dtype, cache):
    """Prompts of ragged lengths are turned, written, cut down, and then every step's token is turned, written, attended with, and
    the cache cut back to its budget: the same state as the 64-bit loops', step after step."""
    from kernels_b200.streaming_attention import paged_attention, paged_cache_evict, paged_cache_write, rotary_embedding

    B, H, H_kv, D, page, M, budget, recent = 3, 4, 2, 64, 16, 8, 64, 8
    gen = torch.Generator().manual_seed(11)
    c = make_cache(B, H_kv, D, page, [M * page] * B, cache)
    c["lens"] = torch.zeros(B, dtype=torch.int32)
    c["weights"], c["row_positions"] = torch.zeros(B, H_kv, M * page), torch.zeros(B, H_kv, M * page, dtype=torch.int32)
    g = cuda(c)
    prompt = torch.tensor([100, 64, 3], dtype=torch.int32)
    inv_freq = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).cuda()
    scales = dict(k_scale=g.get("k_scale"), v_scale=g.get("v_scale"))
    pages = (g["k_pages"], g["v_pages"], g["page_table"])
    at = torch.zeros(B, dtype=torch.int32)
    for step in range(6):
        T = int(prompt.max()) if step == 0 else 1
        q, k, v = (torch.randn(B, h, T, D, generator=gen).to(dtype).cuda() for h in (H, H_kv, H_kv))
        new = prompt if step == 0 else torch.ones(B, dtype=torch.int32)
        positions = (at[:, None] + torch.arange(T, dtype=torch.int32)[None]).cuda()
        q, k = rotary_embedding(q, k, positions[None], inv_freq)
        c["lens"] += new
        g["lens"] += new.cuda()
        paged_cache_write(k, v, *pages, g["lens"], new.cuda(), positions, g["weights"], g["row_positions"], **scales)
        PO.write(k.cpu(), v.cpu(), c["k_pages"], c["v_pages"], c["page_table"], c["lens"], new, positions.cpu(), c["weights"], c["row_positions"],
                 c.get("k_scale"), c.get("v_scale"))
        last = (new.long() - 1).cuda()
        q1 = q[torch.arange(B).cuda(), :, last]
        o, _ = check_attend(c, q1.cpu(), on_gpu=g)
        # weights from the kernel feed both sides, so that rounding cannot tip a choice between two rows
        got = paged_attention(q1, *pages, g["lens"], weights=g["weights"], **scales)
        assert torch.equal(got.cpu().double(), o)
        c["weights"] = g["weights"].cpu()
        paged_cache_evict(*pages, g["lens"], g["weights"], g["row_positions"], budget, recent, **scales)
        PO.evict(c["k_pages"], c["v_pages"], c["page_table"], c["lens"], c["weights"], c["row_positions"], budget, recent, c.get("k_scale"), c.get("v_scale"))
        for n, x in c.items():
            y = g[n].cpu()
            x, y = (t.view(torch.uint8) if t.dtype == F8 else t for t in (x, y))
            assert torch.equal(x, y), (step, n)
        at += new
    assert c["lens"].tolist() == [64, 64, 8]


def test_a_captured_decoding_step_replays():
    from kernels_b200.streaming_attention import paged_attention, paged_cache_evict, paged_cache_write, rotary_embedding

    B, H, H_kv, D, page, M, budget = 2, 8, 2, 128, 16, 40, 600
    start = cuda(make_cache(B, H_kv, D, page, [M * page] * B, BF16))
    inv_freq = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).cuda()
    tokens = [[torch.randn(B, h, 1, D, device="cuda").bfloat16() for h in (H, H_kv, H_kv)] for _ in range(5)]

    def state():
        s = {n: x.clone() for n, x in start.items()}
        s["lens"][:] = torch.tensor([598, 20])
        s["weights"] = torch.rand(B, H_kv, M * page, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
        s["row_positions"] = torch.arange(M * page, dtype=torch.int32, device="cuda").expand(B, H_kv, -1).contiguous()
        s["at"] = s["lens"][:, None].clone()
        return s

    def step(s, q, k, v):
        s["lens"] += 1
        q, k = rotary_embedding(q, k, s["at"][None], inv_freq)
        paged_cache_write(k, v, s["k_pages"], s["v_pages"], s["page_table"], s["lens"], None, s["at"], s["weights"], s["row_positions"])
        o = paged_attention(q[:, :, 0], s["k_pages"], s["v_pages"], s["page_table"], s["lens"], weights=s["weights"])
        paged_cache_evict(s["k_pages"], s["v_pages"], s["page_table"], s["lens"], s["weights"], s["row_positions"], budget, 32)
        s["at"] += 1
        return o

    eager, want = state(), []
    for t in tokens:
        want.append(step(eager, *t))
    s = state()
    fixed = [x.clone() for x in tokens[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(s, *fixed)
    for t, w in zip(tokens, want):
        for x, y in zip(fixed, t):
            x.copy_(y)
        graph.replay()
        assert torch.equal(o, w)
    assert all(torch.equal(s[n], eager[n]) for n in s)


def test_two_streams_at_once():
    """Calls whose workspaces live at the same time on two streams."""
    from kernels_b200.streaming_attention import paged_attention, paged_cache_evict

    made = []
    for seed in (0, 1):
        c = make_cache(2, 2, 128, 64, [4000, 1500], BF16, seed=seed)
        w, pos = make_books(2, 2, c["page_table"].shape[1] * 64, seed=seed)
        made.append((cuda(c), w.cuda(), pos.cuda(), torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()))

    def work(g, w, pos, q):
        g, w, pos = {n: x.clone() for n, x in g.items()}, w.clone(), pos.clone()
        args = (g["k_pages"], g["v_pages"], g["page_table"], g["lens"])
        outs = [paged_attention(q, *args, weights=w)]
        paged_cache_evict(*args, w, pos, 1000, 50)
        outs.append(paged_attention(q, *args, weights=w))
        return outs + [w, pos, *g.values()]

    want = [work(*m) for m in made]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in made], [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = work(*made[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))

def test_lazily_negated_tensors():
    """A tensor whose sign is a mark on it (the imaginary part of a conjugate): new tokens and queries are taken as the numbers that they are, a cache
    like that is refused."""
    from kernels_b200.streaming_attention import paged_attention, paged_cache_evict, paged_cache_write

    def marked(x):
        y = torch.complex(torch.zeros_like(x), -x).conj().imag
        assert y.is_neg() and torch.equal(y, x)
        return y

    c = make_cache(2, 2, 64, 16, [40, 30], F32)
    k, v, q = torch.randn(2, 2, 3, 64), torch.randn(2, 2, 3, 64), torch.randn(2, 4, 64)
    check_write(c, k, v, kg=marked(k.cuda()))
    check_write(c, k, v, vg=marked(v.cuda()))
    g = cuda(c)
    pages = dict(k_pages=g["k_pages"], v_pages=g["v_pages"], page_table=g["page_table"], lens=g["lens"])
    want = paged_attention(q.cuda(), **pages)
    assert torch.equal(paged_attention(marked(q.cuda()), **pages), want)
    w, pos = torch.zeros(2, 2, 48, device="cuda"), torch.zeros(2, 2, 48, dtype=torch.int32, device="cuda")
    for change in (dict(k_pages=marked(g["k_pages"])), dict(v_pages=marked(g["v_pages"])), dict(weights=marked(w))):
        with pytest.raises(AssertionError):
            paged_attention(**(dict(q=q.cuda()) | pages | change))
        with pytest.raises(AssertionError):
            paged_cache_write(**(dict(k=k.cuda(), v=v.cuda()) | pages | change))
        with pytest.raises(AssertionError):
            paged_cache_evict(**(dict(weights=w, row_positions=pos, budget=8) | pages | change))
    f8 = cuda(make_cache(2, 2, 64, 16, [40, 30], F8))
    with pytest.raises(AssertionError):
        paged_attention(q.cuda(), f8["k_pages"], f8["v_pages"], f8["page_table"], f8["lens"], k_scale=marked(f8["k_scale"]), v_scale=f8["v_scale"])


def test_calls_under_whatever_traces_are_refused():
    """What records operators would record nothing of these calls."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from kernels_b200.streaming_attention import paged_attention, paged_cache_evict, paged_cache_write

    g = cuda(make_cache(2, 2, 64, 16, [40, 30], F32))
    pages, q = dict(k_pages=g["k_pages"], v_pages=g["v_pages"], page_table=g["page_table"], lens=g["lens"]), torch.randn(2, 4, 64)
    w, pos = torch.zeros(2, 2, 48, device="cuda"), torch.zeros(2, 2, 48, dtype=torch.int32, device="cuda")
    calls = (lambda x: paged_attention(x, **pages), lambda x: paged_cache_write(x[:, :2, None], x[:, :2, None], **pages) or x,
             lambda x: paged_cache_evict(**pages, weights=w, row_positions=pos, budget=8)[1] + x[0, 0, 0])
    before = {n: x.clone() for n, x in g.items()}
    for call in calls:
        with pytest.raises(RuntimeError, match="trac"):
            torch.jit.trace(call, (q.cuda(),), check_trace=False)
        with pytest.raises(RuntimeError, match="trac"):
            make_fx(call)(q.cuda())
    for call in calls[:2]:  # (no rule for batches of calls; the third has none of a batch's tensors)
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(q.cuda()[None])
    assert all(torch.equal(before[n], g[n]) for n in g)


def test_calls_from_a_compiled_function():
    """A compiled function steps out for these calls: the eager results."""
    from kernels_b200.streaming_attention import paged_attention, paged_cache_evict, paged_cache_write

    c = make_cache(2, 2, 64, 16, [90, 70], F16)
    w, pos = make_books(2, 2, c["page_table"].shape[1] * 16)
    q, k = torch.randn(2, 4, 64).half().cuda(), torch.randn(2, 2, 3, 64).half().cuda()

    def step(g, w, pos, q, k):
        paged_cache_write(k * 2, k, g["k_pages"], g["v_pages"], g["page_table"], g["lens"], weights=w, row_positions=pos)
        o = paged_attention(q * 2, g["k_pages"], g["v_pages"], g["page_table"], g["lens"], weights=w) + 1
        paged_cache_evict(g["k_pages"], g["v_pages"], g["page_table"], g["lens"], w, pos, 50, 4)
        return o

    results = []
    for f in (step, torch.compile(step)):
        g = cuda(c | dict(w=w, pos=pos))
        results.append((f(g, g["w"], g["pos"], q, k), g))
    (a, x), (b, y) = results
    assert torch.equal(a, b) and all(torch.equal(x[n], y[n]) for n in x)


# ---- refusals ------------------------------------------------------------------------------------------------------


def test_refusals():
    from kernels_b200.streaming_attention import paged_attention, paged_cache_evict, paged_cache_write

    g = cuda(make_cache(2, 2, 64, 16, [40, 30], F16))
    f8 = cuda(make_cache(2, 2, 64, 16, [40, 30], F8))
    pages = dict(k_pages=g["k_pages"], v_pages=g["v_pages"], page_table=g["page_table"], lens=g["lens"])
    q, k = torch.zeros(2, 4, 64, dtype=F16, device="cuda"), torch.zeros(2, 2, 3, 64, dtype=F16, device="cuda")
    L = g["page_table"].shape[1] * 16
    w, pos = torch.zeros(2, 2, L, device="cuda"), torch.zeros(2, 2, L, dtype=torch.int32, device="cuda")
    cache_bad = [
        dict(v_pages=g["v_pages"][:1]), dict(v_pages=g["v_pages"].float()), dict(page_table=g["page_table"].long()), dict(page_table=g["page_table"][:1]),
        dict(page_table=g["page_table"][0]), dict(lens=g["lens"].long()), dict(lens=g["lens"][:, None]), dict(lens=g["lens"].cpu()),
        dict(page_table=g["page_table"].cpu()), dict(k_scale=f8["k_scale"], v_scale=f8["v_scale"]), dict(k_pages=f8["k_pages"], v_pages=f8["v_pages"]),
        dict(k_pages=f8["k_pages"], v_pages=f8["v_pages"], k_scale=f8["k_scale"], v_scale=f8["v_scale"].half()),
        dict(k_pages=f8["k_pages"], v_pages=f8["v_pages"], k_scale=f8["k_scale"], v_scale=f8["v_scale"][:, :1]),
        dict(k_pages=g["k_pages"].transpose(2, 3), v_pages=g["v_pages"].transpose(2, 3)), dict(k_pages=g["k_pages"][0], v_pages=g["v_pages"][0]),
    ]
    calls = [
        (paged_attention, dict(q=q), [dict(q=q[:1]), dict(q=q[:, :3]), dict(q=q.float()), dict(q=q[..., :32]), dict(q=q[0]), dict(q=q.cpu()), dict(context_size=0),
                                      dict(back_contexts=-1), dict(weights=w[:, :1]), dict(weights=w[..., 1:]), dict(weights=w.double()),
                                      dict(weights=w.transpose(1, 2)), dict(weights=w.cpu()), dict(weights=w[:1].expand(2, 2, L))]),
        (paged_cache_write, dict(k=k, v=k), [dict(k=k[:1], v=k[:1]), dict(v=k[:, :1]), dict(k=k.float(), v=k.float()), dict(k=k[..., :32], v=k[..., :32]),
                                             dict(new_lens=g["lens"].long()), dict(new_lens=g["lens"][:1]), dict(positions=g["lens"]), dict(weights=w[..., 1:]),
                                             dict(positions=torch.zeros(2, 3, device="cuda")), dict(row_positions=w), dict(v=k.cpu())]),
        (paged_cache_evict, dict(weights=w, row_positions=pos, budget=8), [dict(budget=0), dict(recent=-1), dict(weights=pos), dict(row_positions=w),
                                                                          dict(weights=w[..., :-1]), dict(out=(g["lens"], w)), dict(out=(g["lens"].long(), w, pos)),
                                                                          dict(out=(g["lens"], w[:1], pos))]),
    ]
    before = {n: x.clone() for n, x in g.items()}
    for call, args, bad in calls:
        for change in cache_bad + bad:
            with pytest.raises(AssertionError):
                call(**(pages | args | change))
    # out overlaps in part only
    with pytest.raises((RuntimeError, AssertionError)):
        paged_cache_evict(**pages, weights=w, row_positions=pos, budget=8, out=(g["lens"].clone(), w, pos.clone()))
    for change in (dict(k_pages=g["k_pages"][..., :48], v_pages=g["v_pages"][..., :48], q=q[..., :48]),
                   dict(k_pages=g["k_pages"].double(), v_pages=g["v_pages"].double(), q=q.double())):
        with pytest.raises(RuntimeError, match="unsupported"):
            paged_attention(**(pages | change))
    assert all(torch.equal(before[n], g[n]) for n in g)


def test_written_tensors_that_overlap_themselves_are_refused():
    """One place in memory for several rows, heads or lengths: reading them is fine, writing them would depend on the order."""
    from kernels_b200.streaming_attention import paged_attention, paged_cache_evict, paged_cache_write

    c = make_cache(2, 2, 64, 16, [40, 30], F8)
    g = cuda(c)
    w, pos = torch.zeros(2, 2, 48, device="cuda"), torch.zeros(2, 2, 48, dtype=torch.int32, device="cuda")
    k = torch.randn(2, 2, 3, 64, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda").half()
    pages = {n: g[n] for n in ("k_pages", "v_pages", "page_table", "lens", "k_scale", "v_scale")}
    one = lambda x, d: x.narrow(d, 0, 1).expand(x.shape)  # noqa: E731
    for name in ("k_pages", "v_pages", "k_scale", "v_scale"):
        for d in range(3):
            change = {name: one(g[name], d)}
            assert paged_attention(q, **(pages | change)).shape == q.shape
            with pytest.raises(AssertionError):
                paged_cache_write(k, k, **(pages | change))
            with pytest.raises(AssertionError):
                paged_cache_evict(**(pages | change), weights=w, row_positions=pos, budget=8)
    with pytest.raises(AssertionError):
        paged_cache_evict(**pages, weights=w, row_positions=pos, budget=8, out=(g["lens"][:1].expand(2), w.clone(), pos.clone()))
    # a single page, head or row may have any stride
    small = {n: torch.zeros(1, 1, 1, *s, dtype=t, device="cuda").expand(1, 1, 1, *s) for n, s, t in (("k_pages", (64,), F16), ("v_pages", (64,), F16))}
    small = {n: x.as_strided(x.shape, (0, 0, 0, 1)) for n, x in small.items()}
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    x = torch.randn(1, 1, 1, 64, device="cuda").half()
    paged_cache_write(x, x, **small, page_table=i([[0]]), lens=i([1]))
    assert torch.equal(small["k_pages"], x) and torch.equal(small["v_pages"], x)
