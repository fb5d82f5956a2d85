"""The paged cache of 4 bits: what its store writes, bit by bit, and the attention over it against the same sums in 64 bits."""

import math

import pytest
import torch

from plain import ops_ref as R

DEV = "cuda:0"
gpu = pytest.mark.gpu


def ops():
    from qwen3_runtime_amd.ops.hip import HipOps

    return HipOps()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def codes_of(x):
    """Codes, lowest value and step of every vector of x [..., D], by the definition in csrc/cache4.h."""
    x = x.float()
    low = x.amin(-1, keepdim=True).to(torch.bfloat16)
    span = x.amax(-1, keepdim=True) - low.float()
    step = (span / torch.full_like(span, 15)).to(torch.bfloat16)
    code = torch.where(step > 0, (x - low.float()) / step.float(), 0.0).round().clamp(0, 15).to(torch.uint8)
    step = torch.where(step > 0, step, 0.0)
    broken = ~torch.isfinite(x).all(-1, keepdim=True) | ~torch.isfinite(step)
    low, step = torch.where(broken, float("nan"), low), torch.where(broken, 0.0, step)
    return torch.where(broken, 0, code), low[..., 0], step[..., 0]


def element_places(d):
    """For element e of a key: (byte, shift); of a value of token j of a four: (byte, shift) with 4 * byte + j from the four's start."""
    key = [(e // 2, 4 * (e % 2)) for e in range(d)]
    value = [((e % 16) * (d // 32) + e // 32, 4 * (e // 16 % 2)) for e in range(d)]
    return key, value


def empty_cache(pages, nkv, ps, d, window=None):
    from qwen3_runtime_amd.parts.base import CacheView, GroupView
    from qwen3_runtime_amd.parts.plan import CacheSpec

    t = {"k": torch.zeros(pages, nkv, ps, d // 2, dtype=torch.uint8), "v": torch.zeros(pages, nkv, ps, d // 2, dtype=torch.uint8),
         "steps": torch.zeros(pages, nkv, ps, 4, dtype=torch.bfloat16)}
    t = {n: x.to(DEV) for n, x in t.items()}
    return CacheView(CacheSpec("paged_kv", heads=nkv, head_dim=d, bits=4, window=window), group=GroupView(ps, window, None, None), k=t["k"], v=t["v"], pages=t)


def held(cache, d):
    """(keys, values) [pages, heads, page, D] float32 that the cache holds, element by element."""
    key, value = element_places(d)
    k, v, steps = (cache.pages[n].cpu() for n in ("k", "v", "steps"))
    pages, nkv, ps, _ = k.shape
    ks = torch.stack([k[..., b] >> s & 15 for b, s in key], -1).float()
    fours = v.view(pages, nkv, ps // 4, -1, 4)
    vs = torch.stack([fours[..., b, :] >> s & 15 for b, s in value], -1).reshape(pages, nkv, ps, d).float()
    st = steps.float()
    return st[..., 0:1] + st[..., 1:2] * ks, st[..., 2:3] + st[..., 3:4] * vs


def put(cache, page, off, k, v, d):
    """Keys and values [T, heads, D] into the cache at (page, off), on the host."""
    key, value = element_places(d)
    t = {n: cache.pages[n].cpu() for n in ("k", "v", "steps")}
    pages, nkv, ps, _ = t["k"].shape
    kc, kl, kst = codes_of(k)
    vc, vl, vst = codes_of(v)
    kb, vb = torch.zeros(*k.shape[:2], d // 2, dtype=torch.uint8), torch.zeros(*k.shape[:2], d // 2, dtype=torch.uint8)
    for e in range(d):
        kb[..., key[e][0]] |= kc[..., e] << key[e][1]
        vb[..., value[e][0]] |= vc[..., e] << value[e][1]
    t["k"][page, :, off] = kb
    t["v"].view(pages, nkv, ps // 4, d // 2, 4)[page, :, off // 4, :, off % 4] = vb
    t["steps"][page, :, off] = torch.stack([kl, kst, vl, vst], -1)
    for n in t:
        cache.pages[n].copy_(t[n])


def same(cache, other):
    for n in ("k", "v"):
        assert torch.equal(cache.pages[n].cpu(), other.pages[n].cpu()), n
    # lowest values and steps bit by bit, but for which NaN
    a, b = cache.pages["steps"].cpu(), other.pages["steps"].cpu()
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,nkv,d,ps", [(1, 1, 32, 4), (3, 2, 64, 8), (7, 5, 96, 24), (70, 8, 128, 16), (33, 2, 160, 12), (9, 3, 192, 16), (5, 2, 224, 32), (130, 1, 256, 16)])
def test_store(t, nkv, d, ps, dtype):
    g = gen(t + d)
    pages = -(-t // ps) + 3
    k, v = torch.randn(t, nkv, d, generator=g).to(dtype), (torch.randn(t, nkv, d, generator=g) * 30 + 7).to(dtype)
    k[0, 0] = 0.75             # a vector of one value
    v[t // 2, nkv - 1] *= 1e30
    at = torch.randperm(pages * ps, generator=g)[:t] if t < 20 else torch.arange(t) + 3
    cache, want = empty_cache(pages, nkv, ps, d), empty_cache(pages, nkv, ps, d)
    for c in (cache, want):  # what lies in the other places stays
        for n in ("k", "v"):
            c.pages[n].copy_(torch.randint(256, c.pages[n].shape, generator=gen(1), dtype=torch.uint8))
        c.pages["steps"].copy_(torch.randn(c.pages["steps"].shape, generator=gen(2)).to(torch.bfloat16))
    cache.group.slots = at.to(torch.int32).to(DEV)
    ops().kv_store(k.to(DEV), v.to(DEV), cache)
    put(want, at // ps, at % ps, k, v, d)
    same(cache, want)
    hk, hv = held(cache, d)
    # what is held is off by half a step, and by what rounding the lowest value and the step (twice 2^-8) moves its ends
    for x, h, lo in ((k, hk, 0), (v, hv, 2)):
        st = cache.pages["steps"].cpu().float()[at // ps, :, at % ps]
        off = (h[at // ps, :, at % ps] - x.float()).abs()
        assert bool((off <= 0.5 * st[..., lo + 1: lo + 2] + 15 * 2.0 ** -8 * st[..., lo + 1: lo + 2] + 2.0 ** -8 * st[..., lo: lo + 1].abs() + 1e-30).all())


@gpu
@pytest.mark.parametrize("t", [29, 400])
def test_codes_of_vectors_of_any_magnitude(t):
    """Quotients as a division rounds them: magnitudes from 2^-120 to 2^120, quotients at halves of whole numbers and next to them."""
    g = gen(t)
    nkv, d, ps = 2, 64, 16
    x = torch.randn(2, t, nkv, d, generator=g)
    ties = torch.arange(d) % 31 / 2 + torch.randint(-1, 2, (2, t // 2, nkv, d), generator=g) * 2.0 ** -22
    ties[..., 0], ties[..., 1] = 0.0, 15.0
    x[:, : t // 2] = ties * (1 + torch.randint(0, 128, (2, t // 2, nkv, 1), generator=g) / 128)
    x = x * 2.0 ** torch.randint(-120, 121, (2, t, nkv, 1), generator=g).float()
    cache, want = empty_cache(-(-t // ps), nkv, ps, d), empty_cache(-(-t // ps), nkv, ps, d)
    at = torch.arange(t)
    cache.group.slots = at.to(torch.int32).to(DEV)
    ops().kv_store(x[0].to(DEV), x[1].to(DEV), cache)
    put(want, at // ps, at % ps, x[0], x[1], d)
    same(cache, want)
    qkv = torch.cat([torch.zeros(t, d), x[0].reshape(t, -1), x[1].reshape(t, -1)], 1)  # without a norm or a turn: few tokens by the other kernel
    cache = empty_cache(-(-t // ps), nkv, ps, d)
    cache.group.slots = at.to(torch.int32).to(DEV)
    ops().qk_norm_rope_store(qkv.to(DEV), 1, nkv, d, None, None, 1e-6, None, at.to(torch.int32).to(DEV), cache)
    same(cache, want)


@gpu
def test_store_leaves_out_slots_in_no_page_and_marks_what_is_not_finite():
    t, nkv, d, ps = 9, 2, 128, 16
    k, v = torch.randn(t, nkv, d, generator=gen(1)), torch.randn(t, nkv, d, generator=gen(2))
    k[1, 0, 5], k[2, 1, 127], v[3, 0, 0], v[4, 1, 1], k[5, 0, 0], k[5, 0, 1] = float("nan"), float("inf"), float("-inf"), float("nan"), 3e38, -3e38
    slots = torch.tensor([0, 1, 2, 3, 4, 5, -1, 32, 2 ** 31 - 1], dtype=torch.int32)
    cache, want = empty_cache(2, nkv, ps, d), empty_cache(2, nkv, ps, d)
    cache.group.slots = slots.to(DEV)
    ops().kv_store(k.to(DEV), v.to(DEV), cache)
    put(want, torch.zeros(6, dtype=torch.long), torch.arange(6), k[:6], v[:6], d)
    same(cache, want)
    hk, hv = held(cache, d)
    assert hk[0, 0, 1].isnan().all() and hk[0, 1, 2].isnan().all() and hv[0, 0, 3].isnan().all() and hk[0, 0, 5].isnan().all()
    assert torch.isfinite(hk[0, 0, 0]).all() and torch.isfinite(hv[0, 1, 3]).all()


def case(seqs, nq, nkv, d, ps, dtype, seed=0, window=None, width=0):
    """seqs: [(q_len, kv_len)]. Every place that no sequence has written holds noise between NaN and infinities."""
    from qwen3_runtime_amd.parts.base import StepContext

    g = gen(seed)
    counts = [-(-kv // ps) for _, kv in seqs]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(seqs), max(max(counts), width)), -1, dtype=torch.int32)
    cache = empty_cache(pages, nkv, ps, d, window)
    at = 0
    written = torch.zeros(pages, ps, dtype=torch.bool)
    for s, (_, kv) in enumerate(seqs):
        table[s, : counts[s]] = order[at: at + counts[s]].to(torch.int32)
        at += counts[s]
        pos = torch.arange(kv)
        written[table[s, pos // ps].long(), pos % ps] = True
    for n in ("k", "v"):
        cache.pages[n].copy_(torch.randint(256, cache.pages[n].shape, generator=g, dtype=torch.uint8))
    low, step = -2 - torch.rand(pages, nkv, ps, 2, generator=g), 0.2 + 0.2 * torch.rand(pages, nkv, ps, 2, generator=g)
    steps = torch.stack([low, step], -1).reshape(pages, nkv, ps, 4)
    bad = torch.tensor([float("nan"), float("inf"), float("-inf")])[torch.arange(pages * ps * 4).view(pages, 1, ps, 4) % 3]
    cache.pages["steps"].copy_(torch.where(written[:, None, :, None], steps, bad).to(torch.bfloat16))
    t = sum(q for q, _ in seqs)
    q = torch.randn(t, nq * d, generator=g).to(dtype).to(DEV)
    cu, positions, of = [0], [], []
    for s, (n, kv) in enumerate(seqs):
        cu.append(cu[-1] + n)
        positions += range(kv - n, kv)
        of += [s] * n
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    cache.group.block_table = table.to(DEV)
    ctx = StepContext(ops=None, dtype=dtype, device=torch.device(DEV), num_tokens=t, num_seqs=len(seqs), positions=i32(positions), cu_q=i32(cu),
                      kv_lens=i32([kv for _, kv in seqs]), seq_of_token=i32(of), state_slots=i32([0] * len(seqs)), first_span=i32([0] * len(seqs)),
                      q_lens_host=[n for n, _ in seqs], kv_lens_host=[kv for _, kv in seqs], max_q_len=max(n for n, _ in seqs),
                      max_kv_len=max(kv for _, kv in seqs), groups=[cache.group])
    return q, cache, ctx


def plain(q, cache, ctx, nq, nkv, d, scale, window=None, **more):
    k, v = held(cache, d)
    return R.paged_attention(q.double().cpu(), k.double(), v.double().transpose(2, 3).contiguous(), ctx.cu_q.cpu(), ctx.kv_lens.cpu(),
                             cache.group.block_table.cpu(), cache.group.page_size, nq, nkv, d, scale, window, compute=torch.float64, **more)


def near(got, want, cache):
    """bfloat16: a weight's rounding (2^-8) multiplies step * (n - 8), at most 8 steps; the result's own rounding is 2^-8 of it. In 32
    bits queries and weights are whole, sums of up to 256 products of at most 31 steps by a query of some 4 are off by a few of
    their last places, 2^-24 * 31 * 4 * 16 * step * scale in a score of one standard deviation after another, which is 2e-5 of a weight and of values of 5."""
    top = float(cache.pages["steps"][..., 3].float().nan_to_num(0, 0, 0).max())
    if got.dtype == torch.bfloat16:
        bound = 2.0 ** -8 * 1.01 * (8 * top + want.abs()) + 1e-4
    else:
        bound = torch.full_like(want, 1e-4)
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(off).all() and bool((off <= bound).all()), f"off by {float(off.max())}, {float((off / bound).max())} of the bound"


SHAPES = [
    # (seqs, nq, nkv, d, page)
    ([(1, 1)], 4, 2, 32, 16),
    ([(1, 2), (1, 31), (1, 32), (1, 33), (1, 64), (1, 65)], 6, 2, 32, 8),
    ([(7, 7), (1, 40), (33, 33)], 4, 2, 64, 16),
    ([(5, 37), (1, 17), (2, 95), (24, 24)], 6, 2, 32, 8),
    ([(70, 70)], 5, 1, 96, 24),                       # pages that are no power of two
    ([(3, 130), (64, 64)], 8, 2, 64, 64),
    ([(40, 200), (1, 1000)], 32, 8, 128, 16),         # a portion and a decoded token
    ([(1, 700)], 34, 2, 32, 32),                      # more heads in a group than a tile has rows
    ([(9, 50), (130, 131)], 3, 3, 160, 4),
    ([(20, 131), (150, 300)], 4, 1, 192, 40),
    ([(1, 900), (17, 17)], 16, 1, 224, 16),
    ([(1, 333), (35, 90)], 16, 2, 256, 12),
    ([(300, 1100)], 8, 2, 128, 16),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("splits", [None, 1, 3])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(shape, splits, dtype):
    seqs, nq, nkv, d, ps = SHAPES[shape]
    q, cache, ctx = case(seqs, nq, nkv, d, ps, dtype, seed=shape)
    if splits:
        ctx.scratch["attn_splits"] = splits
    near(ops().paged_attention(q, cache, ctx, nq, nkv, d, d ** -0.5, None), plain(q, cache, ctx, nq, nkv, d, d ** -0.5), cache)


OPTIONS = [{"window": 1}, {"window": 37}, {"window": 50, "keep_first": 3}, {"window": 40, "keep_first": 70}, {"chunk": 48}, {"chunk": 7}, {"softcap": 3.0},
           {"sink": True}, {"window": 33, "keep_first": 5, "sink": True, "softcap": 2.0}]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("splits", [None, 3])
@pytest.mark.parametrize("option", range(len(OPTIONS)))
def test_masks_caps_and_sinks(option, splits, dtype):
    more = dict(OPTIONS[option])
    window = more.pop("window", None)
    nq, nkv, d, ps = 8, 2, 64, 16
    q, cache, ctx = case([(1, 1), (1, 300), (70, 97), (9, 9), (33, 264), (3, 500)], nq, nkv, d, ps, dtype, seed=option, window=window)
    if splits:
        ctx.scratch["attn_splits"] = splits
    want = plain(q, cache, ctx, nq, nkv, d, d ** -0.5, window, **more)
    if window:  # pages that no query sees have been given back
        table = cache.group.block_table.clone()
        for s, (n, kv) in enumerate(zip(ctx.q_lens_host, ctx.kv_lens_host)):
            for p in range(-(-more.get("keep_first", 0) // ps), table.shape[1]):
                if (p + 1) * ps <= kv - n - window + 1:
                    table[s, p] = -1
        cache.group.block_table = table
    near(ops().paged_attention(q, cache, ctx, nq, nkv, d, d ** -0.5, window, **more), want, cache)


FORMS = [(torch.bfloat16, 64, 1, 4), (torch.bfloat16, 64, 2, 4), (torch.bfloat16, 128, 2, 2), (torch.bfloat16, 96, 2, 1), (torch.bfloat16, 160, 1, 4),
         (torch.bfloat16, 256, 1, 2), (torch.bfloat16, 192, 1, 1), (torch.float32, 64, 1, 4), (torch.float32, 32, 1, 2), (torch.float32, 128, 1, 2),
         (torch.float32, 256, 1, 2), (torch.float32, 96, 1, 1)]


@gpu
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("option", [{}, {"window": 37}, {"window": 50, "keep_first": 3}, {"chunk": 48}, {"softcap": 3.0, "sink": True}])
@pytest.mark.parametrize("ps", [16, 12])
@pytest.mark.parametrize("dtype,d,row_tiles,groups", FORMS)
def test_every_split_of_rows_and_keys(dtype, d, row_tiles, groups, ps, option, splits, monkeypatch):
    """Which of them a step takes follows from its sizes; here each has to take lengths that leave bands without rows and groups without keys."""
    from qwen3_runtime_amd.ops.hip import HipOps

    monkeypatch.setattr(HipOps, "choose_attention4_rows", staticmethod(lambda rows, nkv, two: (row_tiles, groups)))
    q, cache, ctx = case([(9, 9), (23, 131), (70, 70), (17, 300), (1, 65), (16 * 64 // 3, 400)], 6, 2, d, ps, dtype, seed=d + groups, window=option.get("window"))
    ctx.scratch["attn_splits"] = splits
    near(ops().paged_attention(q, cache, ctx, 6, 2, d, d ** -0.5, option.get("window"), **{k: v for k, v in option.items() if k != "window"}),
         plain(q, cache, ctx, 6, 2, d, d ** -0.5, **option), cache)


@gpu
@pytest.mark.parametrize("seqs,nkv,form", [([(20, 20)] * 40, 4, (1, 4)), ([(30, 41)] * 60, 4, (2, 4)), ([(64, 70)] * 60, 4, (2, 2)), ([(33, 33)] * 500, 4, (2, 1))])
def test_steps_that_take_each_split_by_their_sizes(seqs, nkv, form):
    from qwen3_runtime_amd.ops.hip import HipOps

    assert HipOps.choose_attention4_rows([2 * n for n, _ in seqs], nkv, True) == form
    q, cache, ctx = case(seqs, 2 * nkv, nkv, 32, 16, torch.bfloat16, seed=len(seqs))
    near(ops().paged_attention(q, cache, ctx, 2 * nkv, nkv, 32, 32 ** -0.5, None), plain(q, cache, ctx, 2 * nkv, nkv, 32, 32 ** -0.5), cache)


def test_how_keys_are_cut():
    """Pieces hold every block of the longest sequence, and are no more than the merge has room for."""
    from qwen3_runtime_amd.ops.hip import HipOps

    choose = HipOps.choose_attention4_piece
    for blocks in ([1], [20], [21], [64] * 8, [500] * 16, [1, 2, 3000], [40] * 300, [100000]):
        for most in (max(blocks), 2 * max(blocks)):
            for keys in (True, False):
                piece = choose(most, blocks, len(blocks), 8, keys)
                assert piece >= 1 and -(-most // piece) <= 1024
    assert choose(16, [16], 1, 8, True) == 16 and choose(128, [76] * 64, 64, 8, True) == 128  # one piece: no merge
    assert choose(1000, [1000], 1, 8, True) == 32 and choose(128, [66] * 8, 8, 8, True) < 32


def test_how_rows_are_split():
    from qwen3_runtime_amd.ops.hip import HipOps

    choose = HipOps.choose_attention4_rows
    assert choose([17], 1, True) == (1, 4) and choose([17], 1, False) == (1, 4)
    for rows, nkv in (([40] * 3000, 8), ([100000], 8), ([24] * 4000, 4), ([17, 90000], 2)):
        for two in (True, False):
            row_tiles, groups = choose(rows, nkv, two)
            assert groups in (1, 2, 4) and row_tiles == (2 if two else 1)
    assert choose([24] * 4000, 4, True) == (2, 4)  # rows that fill one band have no use for a second
    assert choose([24] * 4000, 4, False)[1] == 2


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("seqs", [[(75, 75)], [(4, 75), (1, 75)]])
def test_a_token_takes_nothing_from_keys_it_does_not_see(seqs, value, dtype):
    nq, nkv, d, ps = 4, 2, 64, 16
    q, cache, ctx = case(seqs, nq, nkv, d, ps, dtype, window=40)
    attend = lambda: ops().paged_attention(q, cache, ctx, nq, nkv, d, d ** -0.5, 40)  # noqa: E731
    want, pos = attend(), ctx.positions
    assert torch.isfinite(want).all()
    steps = cache.pages["steps"].clone()
    for at in (0, 33, 37, 74):
        sees = (pos >= at) & (pos - at < 40)
        for which in range(4):
            cache.pages["steps"].copy_(steps)
            for s in range(len(seqs)):
                cache.pages["steps"][int(cache.group.block_table[s, at // ps]), :, at % ps, which] = value
            got = attend()
            assert torch.equal(got[~sees], want[~sees])
            # the tokens that see a NaN are NaN (an infinite key's score is -inf, a weight of 0, where the query's sum is negative)
            assert value == value or got[sees].isnan().all()


@gpu
def test_pages_named_in_the_table_that_are_not_in_the_pool_are_not_read_beyond_it():
    """Entries that no query sees may be anything; a wide table and lengths that end inside a page."""
    q, cache, ctx = case([(1, 50), (20, 70)], 4, 2, 64, 16, torch.bfloat16, window=20, width=9)
    want = ops().paged_attention(q, cache, ctx, 4, 2, 64, 0.125, 20)
    t = cache.group.block_table
    t[0, 0], t[0, 1], t[0, 4:], t[1, 0], t[1, 5:] = 2 ** 30, -(2 ** 30), 2 ** 31 - 1, -7, -(2 ** 31)
    assert torch.equal(ops().paged_attention(q, cache, ctx, 4, 2, 64, 0.125, 20), want)


@gpu
@torch.inference_mode()
def test_a_captured_step_is_the_eager_one():
    """Store and attention in one graph, replayed as the sequences grow; two graphs, one after the other."""
    o, nq, nkv, d, ps = ops(), 8, 2, 128, 16
    q, cache, ctx = case([(1, 100), (1, 700), (1, 17)], nq, nkv, d, ps, torch.bfloat16, width=50)
    k, v = torch.randn(3, nkv, d, generator=gen(5)).to(torch.bfloat16).to(DEV), torch.randn(3, nkv, d, generator=gen(6)).to(torch.bfloat16).to(DEV)
    cache.group.slots = torch.tensor([int(cache.group.block_table[s, (n - 1) // ps]) * ps + (n - 1) % ps for s, n in enumerate(ctx.kv_lens_host)], dtype=torch.int32, device=DEV)
    ctx.kv_lens_host, ctx.max_kv_len = [800] * 3, 800  # a bucket's

    def step():
        o.kv_store(k, v, cache)
        return o.paged_attention(q, cache, ctx, nq, nkv, d, d ** -0.5, None)

    step()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=gen(20 + i)).to(torch.bfloat16))
        k.copy_(torch.randn(k.shape, generator=gen(30 + i)).to(torch.bfloat16))
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, step())
        near(step(), plain(q, cache, ctx, nq, nkv, d, d ** -0.5), cache)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,nq,nkv,d,pairs,norm", [(37, 6, 2, 64, 32, True), (1, 32, 8, 128, 64, True), (31, 4, 2, 96, 48, False), (5, 3, 1, 256, 32, True), (2, 2, 2, 32, None, True),
                                                   (8, 5, 5, 160, 80, False), (100, 8, 2, 128, 64, True), (7, 2, 1, 224, 100, True), (3, 2, 1, 64, None, False)])
def test_norm_rotation_and_store_together(t, nq, nkv, d, pairs, norm, dtype):
    """Queries as with an ordinary cache, and in the cache what the store makes of that one's keys and values."""
    from qwen3_runtime_amd.parts.base import CacheView, GroupView
    from qwen3_runtime_amd.parts.plan import CacheSpec

    o, ps = ops(), 16
    pages = t // ps + 3
    qkv = torch.randn(t, (nq + 2 * nkv) * d + 8, generator=gen(1)).to(dtype).to(DEV)
    qw, kw = (1 + 0.1 * torch.randn(d, generator=gen(2))).to(DEV), (1 + 0.1 * torch.randn(d, generator=gen(3))).to(DEV)
    qw, kw = (qw, kw) if norm else (None, None)
    freq = None if pairs is None else (1e4 ** -(torch.arange(pairs) / pairs)).to(DEV)
    pos, slots = torch.arange(t, dtype=torch.int32, device=DEV) + 1000, torch.arange(5, 5 + t, dtype=torch.int32, device=DEV)
    whole = CacheView(CacheSpec("paged_kv", heads=nkv, head_dim=d), group=GroupView(ps, None, None, slots),
                      k=torch.zeros(pages, nkv, ps, d, dtype=dtype, device=DEV), v=torch.zeros(pages, nkv, d, ps, dtype=dtype, device=DEV))
    cache, want = empty_cache(pages, nkv, ps, d), empty_cache(pages, nkv, ps, d)
    cache.group.slots = slots
    q = o.qk_norm_rope_store(qkv, nq, nkv, d, qw, kw, 1e-6, freq, pos, whole, extra=8)
    assert torch.equal(o.qk_norm_rope_store(qkv, nq, nkv, d, qw, kw, 1e-6, freq, pos, cache, extra=8), q)
    at = slots.cpu().long()
    put(want, at // ps, at % ps, whole.k.cpu()[at // ps, :, at % ps], whole.v.cpu()[at // ps, :, :, at % ps], d)
    same(cache, want)


@gpu
def test_few_tokens_whose_slot_is_in_no_page_store_nothing():
    o, t, nq, nkv, d, ps = ops(), 4, 2, 1, 64, 16
    qkv = torch.randn(t, (nq + 2 * nkv) * d, generator=gen(1)).to(DEV)
    qkv[1, nq * d] = float("nan")
    cache, want = empty_cache(2, nkv, ps, d), empty_cache(2, nkv, ps, d)
    cache.group.slots = torch.tensor([-1, 3, 32, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    o.qk_norm_rope_store(qkv, nq, nkv, d, None, None, 0.0, None, torch.zeros(t, dtype=torch.int32, device=DEV), cache)
    k, v = qkv[1:2, nq * d: (nq + 1) * d].view(1, 1, d).cpu(), qkv[1:2, (nq + 1) * d:].view(1, 1, d).cpu()
    put(want, torch.tensor([0]), torch.tensor([3]), k, v, d)
    same(cache, want)


@gpu
def test_attention_refuses():
    from qwen3_runtime_amd.ops import OpsError

    q, cache, ctx = case([(2, 50)], 4, 2, 64, 16, torch.bfloat16)
    o = ops()
    attend = lambda q=q, cache=cache, d=64, nq=4, scale=0.1, window=None, **more: o.paged_attention(q, cache, ctx, nq, 2, d, scale, window, **more)  # noqa: E731
    attend()
    for bad in (dict(gate=torch.zeros(2, 256, dtype=torch.bfloat16, device=DEV)), dict(value_dim=32), dict(window=4, chunk=4), dict(keep_first=3), dict(scale=float("nan")),
                dict(q=q.half()), dict(softcap=-1.0), dict(window=-3), dict(value_turn=(torch.ones(32, device=DEV), "x"))):
        with pytest.raises(OpsError):
            attend(**bad)
    with pytest.raises(OpsError):
        o.paged_attention(q[:, :96 * 2].contiguous(), cache, ctx, 2, 2, 96, 0.1, None)
    table = cache.group.block_table
    for bad in (table[:, :2].contiguous(), table.repeat(2, 1), table.long()):
        cache.group.block_table = bad
        with pytest.raises(OpsError):
            attend()


@gpu
def test_steps_without_tokens_and_sequences_without_any():
    o = ops()
    q, cache, ctx = case([(0, 40), (2, 50), (0, 0), (20, 33), (0, 9)], 4, 2, 64, 16, torch.bfloat16)
    near(o.paged_attention(q, cache, ctx, 4, 2, 64, 0.125, None), plain(q, cache, ctx, 4, 2, 64, 0.125), cache)
    q, cache, ctx = case([(0, 40), (0, 0)], 4, 2, 64, 16, torch.bfloat16)
    assert o.paged_attention(q, cache, ctx, 4, 2, 64, 0.125, None).shape == (0, 256)
    cache.group.slots = torch.zeros(0, dtype=torch.int32, device=DEV)
    o.kv_store(torch.zeros(0, 2, 64, device=DEV), torch.zeros(0, 2, 64, device=DEV), cache)


@gpu
@pytest.mark.parametrize("seqs", [[(1, 60), (1, 300)], [(40, 60), (1, 300)]])
def test_rows_behind_the_last_sequence_and_neighbours_in_the_cache_stay(seqs):
    """A padded batch: the output has rows for the step's tokens alone, what lies behind them in memory stays, and the cache is only read."""
    nq, nkv, d, ps = 4, 2, 64, 16
    q, cache, ctx = case(seqs, nq, nkv, d, ps, torch.bfloat16)
    before = {n: x.clone() for n, x in cache.pages.items()}
    ctx.scratch["attn_splits"] = 3
    out = ops().paged_attention(q, cache, ctx, nq, nkv, d, d ** -0.5, None)
    assert out.shape == q.shape
    for n, x in cache.pages.items():
        assert torch.equal(x.view(torch.uint8), before[n].view(torch.uint8))


@gpu
def test_a_cache_whose_rows_pass_32_bits_of_bytes():
    """Pages beyond the first 4 GiB of a pool: those go by addresses of 64 bits. Only the pages in the table are written."""
    nq, nkv, d, ps, n = 8, 8, 256, 64, 150
    pages = (1 << 32) // (nkv * ps * d // 2) + 40
    o = ops()
    q, cache, ctx = case([(1, n), (70, n)], nq, nkv, d, ps, torch.bfloat16)
    want = o.paged_attention(q, cache, ctx, nq, nkv, d, d ** -0.5, None)
    table, at = cache.group.block_table.clone(), {}
    big = {name: torch.empty((pages, *x.shape[1:]), dtype=x.dtype, device=DEV) for name, x in cache.pages.items()}
    for i, p in enumerate(sorted(set(table[table >= 0].tolist()))):
        at[p] = pages - 1 - i if i % 2 else i
        for name, x in cache.pages.items():
            big[name][at[p]] = x[p]
    cache.group.block_table = torch.tensor([[at.get(p, -1) for p in row] for row in table.tolist()], dtype=torch.int32, device=DEV)
    cache.pages, cache.k, cache.v = big, big["k"], big["v"]
    got = o.paged_attention(q, cache, ctx, nq, nkv, d, d ** -0.5, None)
    assert torch.equal(got, want)
    # the store, there too
    k, v = torch.randn(3, nkv, d, generator=gen(1)).to(DEV), torch.randn(3, nkv, d, generator=gen(2)).to(DEV)
    cache.group.slots = torch.tensor([(pages - 60) * ps + 1, (pages - 60) * ps + 2, (pages - 61) * ps + 63], dtype=torch.int32, device=DEV)
    o.kv_store(k, v, cache)
    low = empty_cache(2, nkv, ps, d)
    low.group.slots = torch.tensor([ps + 1, ps + 2, 63], dtype=torch.int32, device=DEV)
    o.kv_store(k, v, low)
    for name, x in low.pages.items():
        for p, off in ((1, slice(1, 3)), (0, slice(63, 64))):
            a, b = x[p], big[name][pages - 61 + p]
            if name == "v":
                a, b = (y.reshape(nkv, ps // 4, d // 2, 4) for y in (a, b))
                four, j = off.start // 4, slice(off.start % 4, off.start % 4 + off.stop - off.start)
                assert torch.equal(a[:, four, :, j], b[:, four, :, j])
            else:
                assert torch.equal(a[:, off], b[:, off])


# ---- needs no GPU


def test_spec_of_a_cache_of_4_bits():
    from qwen3_runtime_amd.cache import CacheManager
    from qwen3_runtime_amd.parts.plan import CacheSpec

    spec = CacheSpec("paged_kv", heads=2, head_dim=64, bits=4)
    assert spec.bytes_per_token(2) == 2 * (32 + 32 + 8) == spec.bytes_per_token(4)
    assert spec.group_key() != CacheSpec("paged_kv", heads=2, head_dim=64).group_key()
    cache = CacheManager([spec, CacheSpec("paged_kv", heads=2, head_dim=64)], page_size=8, num_pages=5, max_requests=1, dtype=torch.bfloat16)
    assert [s.dtype for s in cache.groups[0].storage] == [torch.uint8, torch.uint8, torch.bfloat16]
    assert CacheManager.bytes_per_page(cache.specs, 8, 2) == 8 * (144 + 2 * 2 * 64 * 2) and cache.bytes_read([10]) == 10 * (144 + 512)
    cache.admit("a")
    from qwen3_runtime_amd.parts.base import GroupView

    view = cache.view(0, [GroupView(8, None, None, None)] * 2)
    assert view.k.shape == view.v.shape == (5, 2, 8, 32) and view.pages["steps"].shape == (5, 2, 8, 4)
    for bad in (dict(bits=8), dict(bits=4, head_dim=48), dict(bits=4, head_dim=288), dict(bits=4, value_dim=32), dict(kind="state", bits=4)):
        with pytest.raises(ValueError):
            CacheSpec(**{"kind": "paged_kv", "heads": 2, "head_dim": 64, **bad})
    with pytest.raises(ValueError, match="multiple of 4"):
        CacheManager([spec], page_size=6, num_pages=5, max_requests=1)


def test_entry_points_refuse_on_the_host():
    from ctypes import c_int, c_long, c_void_p

    from qwen3_runtime_amd.ops.hip import HipOps, _Attn4Plan, attention4_library

    lib, p = HipOps().lib, c_void_p(1 << 20)  # not read: the sizes are refused
    store = lambda t=1, heads=2, d=64, ps=16, dtype=1, stride=128, k=p: lib.qrt_store4(  # noqa: E731
        k, p, c_int(dtype), c_long(stride), c_long(stride), p, p, p, p, c_long(4), c_int(t), c_int(heads), c_int(d), c_int(ps), None)
    for bad in (dict(t=-1), dict(heads=0), dict(d=48), dict(d=288), dict(d=0), dict(ps=6), dict(ps=0), dict(dtype=2), dict(stride=129), dict(k=c_void_p(8))):
        assert store(**bad) != 0, bad
    lib = attention4_library(64)

    def attend(dtype=1, keys=1, row_tiles=1, page_size=16, num_pages=3, table_width=2, q=1 << 20, **fields):
        a, at = _Attn4Plan(), 1 << 20
        for n, x in dict(dict(num_tiles=1, nq=4, nkv=2, num_seqs=1, piece=1, pieces=1), **fields).items():
            setattr(a, n, x)
        return lib.qrt_attention4(bytes(a), q, at, at, at, at, at, at, at, 0, 0, table_width, num_pages, page_size, 0, 1.0, 0.0, dtype, keys, row_tiles, None)

    for bad in (dict(nq=3), dict(nkv=0), dict(page_size=6), dict(num_pages=0), dict(table_width=0), dict(window=-1), dict(window=2, chunk=2), dict(keep_first=1),
                dict(piece=0), dict(pieces=0), dict(pieces=2), dict(dtype=3), dict(nq=34), dict(keys=0, row_tiles=3), dict(keys=0, row_tiles=2, dtype=0), dict(q=(1 << 20) + 2),
                dict(keys=0, tile_seq=1 << 20)):
        assert attend(**bad) != 0, bad
    assert attend(num_tiles=0) == 0
