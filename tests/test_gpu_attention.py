"""GPU tests of the 4-bit cache and of paged attention against their definitions in 64 bits.

Tolerances. The 4-bit cache is exact: its codes, scales and read-back values are
compared bit for bit. Attention is held, element by element, to

    u_out |ref| + (u_w + u_s) sum_j w_j |v_j| + n 2^-25 max |v|

u_out: half a step of the output type. u_w: half a step of the 16-bit type the
weights are rounded to (bf16 2^-8, fp16 and 4-bit caches 2^-11; the error of the
sum in the denominator is covered by counting it twice). u_s: fp32 arithmetic:
scores have D products and sums of magnitude up to `reach`, exponentials 2.8e-6 <
48 * 2^-24 (a degree-4 polynomial; the special-function unit's 2^-22 is less) and
their argument's rounding, sums n terms: 2^-24 (2 (D + 8) reach + n + 64), in
numerator and denominator alike. The last term is what fp16 weights below its
smallest normal number lose (2^-25 of the largest weight each).
"""
import math
import random

import pytest
import torch

from lmpool_b200 import _capi
from lmpool_b200 import kv_transfer as kt
from lmpool_b200 import attention as at
from oracle import attention_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def bound(want: ref.Attended, dtype, q4: bool, dim: int) -> torch.Tensor:
    u_w = 2 * (2.0 ** -11 if q4 else HALF_STEP[dtype])
    u_s = 2 * 2.0 ** -24 * (2 * (dim + 8) * want.reach + want.keys + 64)
    return HALF_STEP[dtype] * want.out.abs() + (u_w + u_s) * want.mass + want.keys * 2.0 ** -25 * want.top


class Case:
    """A paged cache with its sequences: 16-bit or 4-bit, pages in random places, on the GPU and as 64-bit values."""

    def __init__(self, ctx, heads, kv_heads, dim, page, dtype, q4, q_lens=None, seed=0, spare=3, tail=0, spread=0.4):
        g = torch.Generator().manual_seed(seed)
        self.page, self.dim, self.q4, self.dtype = page, dim, q4, dtype
        need = [-(-c // page) for c in ctx]
        N = sum(need) + spare
        order = torch.randperm(N, generator=g).tolist()
        self.tables = torch.full((len(ctx), max(max(need), 1)), -1, dtype=torch.int32)
        at_ = 0
        for i, n in enumerate(need):
            self.tables[i, :n] = torch.tensor(order[at_:at_ + n], dtype=torch.int32)
            at_ += n
        strength = torch.exp(spread * torch.randn(kv_heads, dim, generator=g))
        rows = [(torch.randn(N, page, kv_heads, dim, generator=g) * strength).to(dtype) for _ in range(2)]
        if q4:
            self.k = torch.zeros(N, page, kv_heads, at.q4_row_bytes(dim), dtype=torch.uint8, device=DEV)
            self.v = torch.zeros_like(self.k)
            slots = torch.arange(N * page, device=DEV)
            at.store_kvcache_q4(rows[0].flatten(0, 1).to(DEV), rows[1].flatten(0, 1).to(DEV), self.k, self.v, slots, page)
        else:
            self.k, self.v = rows[0].to(DEV), rows[1].to(DEV)
        self.ctx = torch.tensor(ctx, dtype=torch.int32)
        self.q_lens = q_lens
        self.cu = None
        T = len(ctx)
        if q_lens is not None:
            starts = [0]
            for q in q_lens:
                starts.append(starts[-1] + q)
            self.cu = torch.tensor(starts, dtype=torch.int32)
            T = starts[-1]
        self.q = torch.randn(T + tail, heads, dim, generator=g).to(dtype)

    def values(self):
        if self.q4:
            return ref.q4_cache_rows(self.k.cpu()), ref.q4_cache_rows(self.v.cpu())
        return self.k.cpu().double(), self.v.cpu().double()

    def call(self, **kw):
        f = at.paged_attention_q4 if self.q4 else at.paged_attention
        return f(self.q.to(DEV), self.k, self.v, self.tables.to(DEV), self.ctx.to(DEV), self.page,
                 cu_seqlens_q=None if self.cu is None else self.cu.to(DEV), **kw)

    def want(self, **kw):
        k, v = self.values()
        return ref.attention(self.q, k, v, self.tables, self.ctx, self.cu, **kw)

    def check(self, **kw):
        got = self.call(**kw)
        kt.check_device_status(0)
        want = self.want(**kw)
        err = (got.cpu().double() - want.out).abs()
        lim = bound(want, self.dtype, self.q4, self.dim)
        worst = (err / lim.clamp(min=1e-30)).max().item() if err.numel() else 0.0
        assert not err.isnan().any() and (err <= lim).all(), f"worst error is {worst:.3g} of its bound"
        return got


# ----------------------------------------------------------------------------------------------
# 4-bit rows
# ----------------------------------------------------------------------------------------------

def _rows(T, H, D, dtype, seed):
    """Rows of every kind: normal, tiny, large, constant, zero, with exact ties, with numbers that are not finite."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, D, generator=g) * torch.exp(2 * torch.randn(T, H, 1, generator=g))
    for t in range(T):
        kind = t % 8
        if kind == 1:
            x[t] *= 2.0 ** -12
        elif kind == 2:
            x[t] = x[t].clamp(-4, 4) * 900
        elif kind == 3:
            x[t] = 0.0
        elif kind == 4:     # ties: amax 6 s with s = 1, elements on every border
            ties = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6])
            x[t] = ties.repeat(D // 16) * 2.0 ** (t % 5 - 2)
        elif kind == 5:     # amax / 6 halfway between two scales: 6 * 1.0625 * 2^e
            x[t] = 6 * 1.0625 * 2.0 ** (t % 7 - 3) * torch.linspace(-1, 1, D)
        elif kind == 6 and D >= 32:
            x[t, 0, 3] = math.inf
            x[t, -1, 17] = math.nan
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,D,page", [(1, 1, 16, 16), (17, 3, 64, 16), (40, 2, 128, 32), (33, 1, 80, 48), (9, 8, 256, 16)])
def test_q4_rows_are_those_of_the_definition(require_gpu, dtype, T, H, D, page):
    N = -(-T // page) + 2
    key, value = _rows(T, H, D, dtype, 1), _rows(T, H, D, dtype, 2)
    slots = torch.randperm(N * page, generator=torch.Generator().manual_seed(3))[:T]
    slots[5::6] = -1
    before = torch.randint(0, 256, (2, N, page, H, at.q4_row_bytes(D)), generator=torch.Generator().manual_seed(4)).to(torch.uint8)
    kc, vc = before[0].to(DEV), before[1].to(DEV)
    at.store_kvcache_q4(key.to(DEV), value.to(DEV), kc, vc, slots.to(DEV), page)
    kt.check_device_status(0)
    for rows, cache, got in ((key, before[0], kc), (value, before[1], vc)):
        for t in range(T):
            if slots[t] >= 0:
                for h in range(H):
                    ref.q4_write(cache, int(slots[t]), h, *ref.q4_encode_row(rows[t, h]))
        # A tiny negative number keeps its sign (-0) in both; groups of scale 0 hold codes of 0.
        wrong = (got.cpu() != cache).nonzero().tolist()
        assert not wrong, f"{len(wrong)} bytes differ, the first at {wrong[:4]}"
    k_back, v_back = at.load_kvcache_q4(kc, vc, slots.to(DEV), page, dtype=dtype)
    for back, cache in ((k_back, kc.cpu()), (v_back, vc.cpu())):
        for t in range(T):
            for h in range(H):
                want = ref.q4_read(cache, int(slots[t]), h) if slots[t] >= 0 else [0.0] * D
                assert torch.equal(back[t, h].cpu().double().nan_to_num(7e7), torch.tensor(want, dtype=torch.float64).nan_to_num(7e7))


def test_q4_scales_shift_the_range(require_gpu):
    T, H, D, page = 16, 2, 64, 16
    x = (torch.randn(T, H, D, generator=torch.Generator().manual_seed(5)) * 2.0 ** -14).to(torch.bfloat16)
    kc = torch.zeros(2, page, H, at.q4_row_bytes(D), dtype=torch.uint8, device=DEV)
    vc = torch.zeros_like(kc)
    slots = torch.arange(T, device=DEV)
    at.store_kvcache_q4(x.to(DEV), (x.float() * 2 ** 30).to(x.dtype).to(DEV), kc, vc, slots, page, k_scale=2.0 ** -14, v_scale=2.0 ** 16)
    k, v = at.load_kvcache_q4(kc, vc, slots, page, k_scale=2.0 ** -14, v_scale=2.0 ** 16)
    for t in range(T):
        for h in range(H):
            want = torch.tensor(ref.q4_decode(*ref.q4_encode_row(x[t, h].double() * 2.0 ** 14)), dtype=torch.float64)
            assert torch.equal(k[t, h].cpu().double(), want * 2.0 ** -14)
            assert torch.equal(v[t, h].cpu().double(), want * 2.0 ** 16)


def test_q4_rows_beyond_fp32_saturate(require_gpu):
    """Finite elements that k_scale or v_scale below 1 lifts out of fp32's range are held at the largest value, as any that
    are too large; groups with an infinity or a NaN still read back as NaN."""
    T, H, D, page = 4, 1, 64, 16
    x = torch.randn(T, H, D, generator=torch.Generator().manual_seed(26)).to(torch.bfloat16)
    x[0] *= 2.0 ** 125
    x[1, 0, 5] = -2.0 ** 127
    x[2, 0, 20] = torch.finfo(torch.bfloat16).max
    x[2, 0, 50] = math.inf
    x[3, 0, 3] = math.nan
    kc = torch.zeros(1, page, H, at.q4_row_bytes(D), dtype=torch.uint8, device=DEV)
    vc = torch.zeros_like(kc)
    at.store_kvcache_q4(x.to(DEV), x.to(DEV), kc, vc, torch.arange(T, device=DEV), page, k_scale=0.5, v_scale=2.0 ** -64)
    kt.check_device_status(0)
    for cache, scale in ((kc, 0.5), (vc, 2.0 ** -64)):
        want = torch.zeros(1, page, H, at.q4_row_bytes(D), dtype=torch.uint8)
        for t in range(T):
            ref.q4_write(want, t, 0, *ref.q4_encode_row(x[t, 0].double() / scale))
        assert torch.equal(cache.cpu(), want)


def test_q4_strided_rows_and_views_of_a_stacked_cache(require_gpu):
    """Rows cut out of a fused projection, a cache that is one layer of [2, L, N, ...], and a slot list with gaps."""
    T, H, D, page, L, N = 21, 2, 64, 16, 3, 4
    qkv = torch.randn(T, 5 * H, D, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    cache = torch.zeros(2, L, N, page, H, at.q4_row_bytes(D), dtype=torch.uint8, device=DEV)
    slots = torch.randperm(N * page, generator=torch.Generator().manual_seed(7))[:2 * T].to(DEV)[::2]
    dev = qkv.to(DEV)
    at.store_kvcache_q4(dev[:, 2 * H:3 * H], dev[:, 4 * H:], cache[0, 1], cache[1, 1], slots, page)
    kt.check_device_status(0)
    want = torch.zeros(2, N, page, H, at.q4_row_bytes(D), dtype=torch.uint8)
    for t in range(T):
        for h in range(H):
            ref.q4_write(want[0], int(slots[t]), h, *ref.q4_encode_row(qkv[t, 2 * H + h]))
            ref.q4_write(want[1], int(slots[t]), h, *ref.q4_encode_row(qkv[t, 4 * H + h]))
    assert torch.equal(cache[:, 1].cpu(), want) and int(cache[:, 0].sum()) == 0 and int(cache[:, 2].sum()) == 0


def test_q4_bad_slots_are_flagged_and_skipped(require_gpu):
    T, H, D, page = 4, 1, 32, 16
    x = torch.ones(T, H, D, dtype=torch.float16, device=DEV)
    kc = torch.zeros(2, page, H, at.q4_row_bytes(D), dtype=torch.uint8, device=DEV)
    vc = torch.zeros_like(kc)
    slots = torch.tensor([0, 32, -5, -1], device=DEV)
    at.store_kvcache_q4(x, x, kc, vc, slots, page)
    with pytest.raises(_capi.KvxError, match="slot_mapping"):
        kt.check_device_status(0)
    k, _ = at.load_kvcache_q4(kc, vc, slots, page, dtype=torch.float16)
    with pytest.raises(_capi.KvxError, match="slot_mapping"):
        kt.check_device_status(0)
    # 1 / 6 lies between the scales 10/64 and 11/64 and nearer the second: 6 * 11/64 = 1.03125 is what is kept of 1.
    assert k[0].eq(1.03125).all() and k[1:].eq(0).all()
    assert int((kc != 0).sum()) == D // 2 + D // 16


# ----------------------------------------------------------------------------------------------
# Attention
# ----------------------------------------------------------------------------------------------

TYPES = [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True), (torch.float16, True)]
IDS = ["bf16", "fp16", "bf16-q4", "fp16-q4"]


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,page,window,sinks", [
    (4, 4, 16, None, 0), (6, 2, 32, None, 0), (8, 1, 16, 24, 4), (16, 1, 48, 40, 1), (10, 2, 16, 7, 0), (32, 1, 16, 100, 70)])
def test_decode(require_gpu, dtype, q4, dim, heads, kv_heads, page, window, sinks):
    case = Case([1, 2, 15, 16, 17, 63, 65, 130, 0, 257], heads, kv_heads, dim, page, dtype, q4, seed=heads + dim)
    case.check(window=window, sinks=sinks)


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 3), (300, 20)])
def test_long_decode_is_split_over_the_keys(require_gpu, dtype, q4, window, sinks):
    case = Case([2100, 3], 4, 1, 128, 16, dtype, q4, seed=9)
    case.check(window=window, sinks=sinks)


@pytest.mark.parametrize("page", [1, 3, 8, 24, 100])
def test_pages_of_any_size(require_gpu, page):
    case = Case([1, 37, 101, 250], 8, 2, 128, page, torch.bfloat16, False, seed=page)
    case.check(window=90, sinks=5)
    case = Case([30, 101], 4, 2, 64, page, torch.float16, False, q_lens=[30, 80], seed=page)
    case.check(window=17, sinks=2)


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 128), (8, 1, 64), (7, 1, 128), (2, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3), (64, 70), (1, 0)])
def test_several_tokens_of_a_sequence(require_gpu, dtype, q4, heads, kv_heads, dim, window, sinks):
    """Drafted tokens, chunks of prompts, empty sequences, and tokens that stand before the context (no key: zeros)."""
    case = Case([9, 5, 40, 3, 0, 70], heads, kv_heads, dim, 16, dtype, q4, q_lens=[3, 5, 1, 6, 0, 4], seed=heads)
    got = case.check(window=window, sinks=sinks)
    assert got[9:12].eq(0).all()          # sequence 3: six tokens on a context of three


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 128), (2, 2, 64), (5, 1, 128)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (33, 2), (150, 20)])
def test_prompts(require_gpu, dtype, q4, heads, kv_heads, dim, window, sinks):
    case = Case([200, 331, 64], heads, kv_heads, dim, 32, dtype, q4, q_lens=[200, 131, 64], seed=dim + heads)
    case.check(window=window, sinks=sinks)


@pytest.mark.parametrize("heads,kv_heads", [(48, 1), (71, 1), (256, 1)])
@pytest.mark.parametrize("q_lens", [None, [3, 1]])
def test_many_query_heads_on_one_kv_head(require_gpu, heads, kv_heads, q_lens):
    case = Case([33, 200], heads, kv_heads, 128, 16, torch.bfloat16, False, q_lens=q_lens, seed=heads)
    case.check()


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
def test_a_chunk_on_a_long_context(require_gpu, dtype, q4):
    case = Case([1500], 4, 1, 128, 64, dtype, q4, q_lens=[70], seed=5)
    case.check()
    case.check(window=700, sinks=4)


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
@pytest.mark.parametrize("q_lens", [None, [4, 3], [70, 90]], ids=["decode", "draft", "prompt"])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(require_gpu, dtype, q4, q_lens):
    """Infinite and NaN keys and values outside a row's window, behind its position and behind the context leave that
    row's result as it is; rows that see them follow the formula."""
    case = Case([100, 120], 4, 1, 64, 16, dtype, q4, q_lens=q_lens, seed=3)
    window, sinks = 20, 2
    clean = case.call(window=window, sinks=sinks)
    page_of = lambda s, j: (int(case.tables[s, j // 16]), j % 16)  # noqa: E731
    hit = []
    for s, j, what in ((0, 30, math.nan), (0, 97, math.inf), (1, 60, -math.inf), (1, 118, math.nan)):
        blk, off = page_of(s, j)
        row = torch.full((1, 1, 64), what, dtype=dtype, device=DEV)
        slot = torch.tensor([blk * 16 + off], device=DEV)
        (at.store_kvcache_q4 if q4 else at.store_kvcache)(row, row, case.k, case.v, slot, 16)
        hit.append((s, j))
    # Behind each context: the rest of its last page.
    for s, c in ((0, 100), (1, 120)):
        blk, off = page_of(s, c - 1)
        if not q4:
            case.k[blk, off + 1:] = math.nan
            case.v[blk, off + 1:] = math.inf
    got = case.call(window=window, sinks=sinks)
    kt.check_device_status(0)
    starts = [0, 1, 2] if q_lens is None else case.cu.tolist()
    saw = kept = 0
    for s, c in ((0, 100), (1, 120)):
        n = starts[s + 1] - starts[s]
        for t in range(n):
            p = c - n + t
            sees = any(s == a and j <= p and (p - j < window or j < sinks) for a, j in hit)
            row = got[starts[s] + t]
            if sees:
                saw += 1
                assert not row.isfinite().all()
            else:
                kept += 1
                assert row.isfinite().all()
                # the rare path sums in another order: both are within the bound of the exact result, so 2 bounds apart
                assert (row.float() - clean[starts[s] + t].float()).abs().max() < 0.05
    assert saw and (kept or q_lens is None or q_lens == [4, 3])


@pytest.mark.parametrize("q4", [False, True])
def test_query_strides_and_given_output(require_gpu, q4):
    """Queries cut out of a fused projection, an output with gaps between its rows."""
    case = Case([40, 90], 4, 2, 64, 16, torch.bfloat16, q4, seed=8)
    want = case.check()
    fused = torch.zeros(2, 8, 64, dtype=torch.bfloat16, device=DEV)
    fused[:, 2:6] = case.q.to(DEV)
    buf = torch.full((2, 6, 80), 3.0, dtype=torch.bfloat16, device=DEV)
    out = buf[:, 1:5, 8:72]
    f = at.paged_attention_q4 if q4 else at.paged_attention
    res = f(fused[:, 2:6], case.k, case.v, case.tables.to(DEV), case.ctx.to(DEV), 16, out=out)
    assert res.data_ptr() == out.data_ptr() and torch.equal(res, want)
    assert buf[:, 0].eq(3).all() and buf[:, 5].eq(3).all() and buf[:, :, :8].eq(3).all() and buf[:, :, 72:].eq(3).all()
    # queries at an address that no 16-byte load can start at
    odd = torch.zeros(2 * 4 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(2, 4, 64)
    odd.copy_(case.q.to(DEV))
    assert torch.equal(f(odd, case.k, case.v, case.tables.to(DEV), case.ctx.to(DEV), 16), want)


@pytest.mark.parametrize("q_lens", [None, [40, 70]], ids=["decode", "prompt"])
def test_dimensions_of_one_entry_may_have_any_stride(require_gpu, q_lens):
    """One kv head, one page, one token a page: the stride of such a dimension means nothing."""
    for ctx, page, pages in (([40, 90], 16, None), ([40, 90], 1, None), ([40, 90], 96, 1)):
        case = Case(ctx, 4, 1, 64, page, torch.bfloat16, False, q_lens=q_lens, seed=8)
        if pages == 1:                      # both sequences on the same page
            case.k, case.v, case.tables = case.k[:1].clone(), case.v[:1].clone(), torch.zeros(2, 1, dtype=torch.int32)
        want = case.check()
        shape, size = case.k.shape, case.k.numel()
        odd = [1 if n == 1 else st for n, st in zip(shape, case.k.stride())]
        f = lambda x: torch.as_strided(x.clone(), shape, odd)  # noqa: E731
        assert f(case.k).numel() == size
        got = at.paged_attention(case.q.to(DEV), f(case.k), f(case.v), case.tables.to(DEV), case.ctx.to(DEV), page,
                                 cu_seqlens_q=None if case.cu is None else case.cu.to(DEV))
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
@pytest.mark.parametrize("q_len", [0, 5, 40])
def test_short_contexts_in_wide_tables(require_gpu, dtype, q4, q_len):
    """Tables wide enough for long contexts: most splits have no keys."""
    ctx = [40, 3, 700]
    case = Case(ctx, 4, 1, 64, 16, dtype, q4, q_lens=[min(q_len, c) for c in ctx] if q_len else None, seed=15)
    case.tables = torch.cat((case.tables, torch.full((3, 3000), -1, dtype=torch.int32)), 1)
    case.check()
    case.check(window=9, sinks=1)


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("most", [3, 60])
def test_many_ragged_sequences(require_gpu, q4, most):
    """More sequences than a warp has lanes, many of them without tokens, some without a context."""
    rng = random.Random(most)
    ctx = [rng.choice([0, 1, rng.randint(1, 60), rng.randint(1, 200)]) for _ in range(75)]
    q_lens = [min(c, rng.choice([0, 1, rng.randint(0, most)])) for c in ctx]
    q_lens[40] = most                                   # more tokens than its context may hold
    case = Case(ctx, 4, 2, 64, 16, torch.float16, q4, q_lens=q_lens, seed=16)
    case.check()
    case.check(window=11, sinks=2)


def test_cache_orders(require_gpu):
    """A cache whose heads lie before its slots, and one layer of a stacked cache."""
    case = Case([40, 90], 4, 2, 64, 16, torch.float16, False, seed=8)
    want = case.check()
    for make in (lambda x: x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3),
                 lambda x: torch.stack((x, x * 0), 1)[:, 0]):
        got = at.paged_attention(case.q.to(DEV), make(case.k), make(case.v), case.tables.to(DEV), case.ctx.to(DEV), 16)
        assert torch.equal(got, want)


@pytest.mark.parametrize("q_lens", [[3, 2], [60, 40]])
@pytest.mark.parametrize("ctx", [[30, 20], [3000, 2500]])
def test_rows_behind_the_last_sequence_are_left(require_gpu, q_lens, ctx):
    ctx = [max(c, q) for c, q in zip(ctx, q_lens)]
    case = Case(ctx, 4, 2, 64, 16, torch.float16, False, q_lens=q_lens, tail=5, seed=4)
    out = torch.full(case.q.shape, 7.0, dtype=torch.float16, device=DEV)
    case.call(out=out)
    assert out[sum(q_lens):].eq(7).all() and not out[:sum(q_lens)].eq(7).all()
    n = sum(q_lens)
    lim = bound(want := case.want(), case.dtype, False, 64)
    assert ((out[:n].cpu().double() - want.out[:n]).abs() <= lim[:n]).all()


def test_scale(require_gpu):
    case = Case([70], 4, 4, 64, 16, torch.float16, False, seed=2)
    case.check(scale=0.37)
    q4 = Case([70], 4, 4, 64, 16, torch.bfloat16, True, seed=2)
    a = q4.call(scale=0.25)
    b = q4.call(scale=0.125, k_scale=2.0, v_scale=4.0)
    assert torch.equal(a.float() * 4, b.float())


def test_queries_of_any_size_on_a_4bit_cache(require_gpu):
    """bf16 queries reach past fp16's range: rows are brought into it by powers of two, exactly."""
    case = Case([50], 4, 1, 128, 16, torch.bfloat16, True, seed=6)
    base = case.q.clone()
    for e in (-40, -20, 17, 60):
        case.q = base * 2.0 ** e
        case.check(scale=128 ** -0.5 * 2.0 ** -e)
    case.q = base * torch.tensor([2.0 ** -30, 1.0, 2.0 ** 20, 0.0])[None, :, None].to(torch.bfloat16)
    got = case.call()
    assert got.isfinite().all()


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("q_lens", [None, [6, 3], [90, 30]])
def test_bad_pages_and_lengths_are_flagged(require_gpu, q4, q_lens):
    case = Case([100, 40], 4, 1, 64, 16, torch.float16, q4, q_lens=q_lens, seed=1)
    good = case.call()
    kt.check_device_status(0)
    for bad in (-1, case.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        keep = int(case.tables[0, 2])
        case.tables[0, 2] = bad
        got = case.call()
        with pytest.raises(_capi.KvxError, match="block id"):
            kt.check_device_status(0)
        cut = 1 if q_lens is None else q_lens[0]
        assert torch.equal(got[cut:], good[cut:]) and got.isfinite().all()
        case.tables[0, 2] = keep
    ctx = case.ctx.clone()
    for bad in (-3, case.tables.shape[1] * 16 + 1, 2 ** 31 - 1, -2 ** 31):
        case.ctx[1] = bad
        got = case.call()
        with pytest.raises(_capi.KvxError, match="length"):
            kt.check_device_status(0)
        cut = 1 if q_lens is None else q_lens[0]
        assert torch.equal(got[:cut], good[:cut])
    case.ctx = ctx
    if q_lens is not None:
        for cu in ([0, 200, sum(q_lens)], [0, -5, 3], [5, 3, 9], [0, 4, 2 ** 31 - 1]):
            case.cu = torch.tensor(cu, dtype=torch.int32)
            case.call()
            with pytest.raises(_capi.KvxError, match="length"):
                kt.check_device_status(0)


def test_nothing_to_do(require_gpu):
    case = Case([5], 2, 1, 64, 16, torch.float16, False, q_lens=[0], seed=1)
    assert case.call().shape == (0, 2, 64)
    none = torch.empty(0, 2, 64, dtype=torch.float16, device=DEV)
    got = at.paged_attention(none, case.k, case.v, torch.empty(0, 3, dtype=torch.int32, device=DEV),
                             torch.empty(0, dtype=torch.int32, device=DEV), 16)
    assert got.shape == (0, 2, 64)
    empty = torch.empty(2, 0, dtype=torch.int32, device=DEV)       # no page at all: no key
    got = at.paged_attention(torch.ones(2, 2, 64, dtype=torch.float16, device=DEV), case.k, case.v, empty,
                             torch.zeros(2, dtype=torch.int32, device=DEV), 16)
    assert got.eq(0).all()
    kt.check_device_status(0)


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("q_lens", [None, [4, 4, 4], [100, 60, 30]])
def test_captured_and_replayed_with_other_lengths(require_gpu, q4, q_lens):
    """A captured call reads lengths, tables and rows on the device; two graphs and an eager call do not share scratch."""
    a = Case([900, 120, 40], 4, 1, 128, 16, torch.bfloat16, q4, q_lens=q_lens, seed=11)
    b = Case([900, 700, 30], 4, 1, 128, 16, torch.bfloat16, q4, q_lens=q_lens, seed=12)
    f = at.paged_attention_q4 if q4 else at.paged_attention
    graphs = []
    for case in (a, b):
        st = dict(q=case.q.to(DEV), table=case.tables.to(DEV), ctx=case.ctx.to(DEV),
                  cu=None if case.cu is None else case.cu.to(DEV))
        run = lambda case=case, st=st: f(st["q"], case.k, case.v, st["table"], st["ctx"], 16, cu_seqlens_q=st["cu"])  # noqa: E731
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            st["out"] = run()
        graphs.append((graph, st, run))
    streams = [torch.cuda.Stream(DEV) for _ in graphs]
    for _ in range(3):
        for (graph, st, run), s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream(DEV))
            with torch.cuda.stream(s):
                graph.replay()
        eager = graphs[0][2]()
    torch.cuda.synchronize()
    assert torch.equal(eager, graphs[0][1]["out"])
    for graph, st, run in graphs:
        assert torch.equal(st["out"], run())
    graph, st, run = graphs[0]
    st["ctx"].copy_(torch.tensor([500, 119, 33], dtype=torch.int32))
    st["q"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(st["out"], run())
    kt.check_device_status(0)


def test_on_another_stream(require_gpu):
    case = Case([300, 80], 4, 1, 128, 16, torch.bfloat16, False, seed=13)
    want = case.call()
    torch.cuda.synchronize()
    s = torch.cuda.Stream(DEV)
    q, tables, ctx = case.q.to(DEV), case.tables.to(DEV), case.ctx.to(DEV)
    s.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(s):
        got = at.paged_attention(q, case.k, case.v, tables, ctx, 16)
    s.synchronize()
    assert torch.equal(got, want)


def test_repeated_calls_give_the_same_bits(require_gpu):
    for q_lens in (None, [5, 5], [130, 70]):
        for dtype, q4 in TYPES:
            case = Case([2000, 333], 8, 2, 128, 16, dtype, q4, q_lens=q_lens, seed=14)
            first = case.call(window=900, sinks=4)
            for _ in range(3):
                assert torch.equal(first, case.call(window=900, sinks=4))


@pytest.mark.parametrize("q4", [False, True])
def test_store_move_and_attend_together(require_gpu, q4):
    """As a server uses them: rows stored as they come, pages moved to other places by the block mover, the tables
    rewritten, more rows stored, attention after each step against all rows so far."""
    H, heads, D, page, N, L = 2, 8, 64, 16, 24, 2
    g = torch.Generator().manual_seed(20)
    row = at.q4_row_bytes(D) if q4 else D
    cache = torch.zeros(2, L, N, page, H, row, dtype=torch.uint8 if q4 else torch.bfloat16, device=DEV)
    store = at.store_kvcache_q4 if q4 else at.store_kvcache
    attend = at.paged_attention_q4 if q4 else at.paged_attention
    table = [5, 1, 7, 20]
    rows = torch.randn(2, L, 60, H, D, generator=g).to(torch.bfloat16)
    ctx = 0
    for step, n in enumerate((33, 1, 1, 9, 5)):
        pos = torch.arange(ctx, ctx + n)
        slots = (torch.tensor(table)[pos // page] * page + pos % page).to(DEV)
        q = torch.randn(n, heads, D, generator=g).to(torch.bfloat16)
        for layer in range(L):
            new = rows[:, layer, ctx:ctx + n].to(DEV)
            store(new[0], new[1], cache[0, layer], cache[1, layer], slots, page)
        ctx += n
        if step == 1:
            kt.move_blocks(cache, L, table, [2, 9, 11, 0])
            table = [2, 9, 11, 0]
        for layer in range(L):
            tables = torch.tensor([table], dtype=torch.int32)
            got = attend(q.to(DEV), cache[0, layer], cache[1, layer], tables.to(DEV),
                         torch.tensor([ctx], dtype=torch.int32, device=DEV), page,
                         cu_seqlens_q=torch.tensor([0, n], dtype=torch.int32, device=DEV), window=25, sinks=2)
            kt.check_device_status(0)
            # from the rows themselves, in order: what the pages hold is what was stored
            kv = rows[:, layer, :ctx].double()
            if q4:
                kv = torch.tensor([[[ref.q4_decode(*ref.q4_encode_row(kv[w, t, h])) for h in range(H)] for t in range(ctx)]
                                   for w in range(2)], dtype=torch.float64)
            want = ref.attention(q, kv[0][:, None], kv[1][:, None], [list(range(ctx))], [ctx], [0, n], window=25, sinks=2)
            err = (got.cpu().double() - want.out).abs()
            assert (err <= bound(want, torch.bfloat16, q4, D)).all()


def test_random_cases(require_gpu):
    """Geometries drawn over the whole range of small sizes, every mask and type."""
    rng = random.Random(7)
    for i in range(40):
        dtype, q4 = rng.choice(TYPES)
        kv_heads = rng.choice([1, 2, 3])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 12])
        page = rng.choice([16, 32, 64, 80]) if q4 else rng.choice([1, 4, 16, 17, 64])
        n = rng.randint(1, 4)
        ctx = [rng.choice([0, 1, rng.randint(1, 40), rng.randint(1, 400)]) for _ in range(n)]
        q_lens = rng.choice([None, [rng.randint(0, max(1, min(c, 9))) for c in ctx], [rng.randint(0, c) for c in ctx]])
        window = rng.choice([None, rng.randint(1, 20), rng.randint(1, 300)])
        sinks = rng.choice([0, 1, 5, 40]) if window else 0
        case = Case(ctx, heads, kv_heads, rng.choice([64, 128]), page, dtype, q4, q_lens=q_lens, seed=100 + i)
        case.check(window=window, sinks=sinks)


# ----------------------------------------------------------------------------------------------
# Many items a CTA
# ----------------------------------------------------------------------------------------------

def attended64(case: Case, window=None, sinks=0) -> ref.Attended:
    """ref.attention for sizes that a loop over rows is too slow for: the same in 64 bits, a sequence at a time. What a
    row does not see counts nowhere, whatever it is; an infinite or NaN value that it sees decides its element."""
    k_all, v_all = (x.to(DEV) for x in case.values())
    q_all = case.q.to(DEV).double()
    T, Hq, D = q_all.shape
    H, page = k_all.shape[2], case.page
    out, mass = torch.zeros_like(q_all), torch.zeros_like(q_all)
    reach, keys, top = 0.0, 0, 0.0
    cu = case.cu.tolist() if case.cu is not None else list(range(len(case.ctx) + 1))
    for s, c in enumerate(case.ctx.tolist()):
        n = cu[s + 1] - cu[s]
        if n == 0 or c == 0:
            continue
        j = torch.arange(c)
        blocks, offs = case.tables[s].long()[j // page].to(DEV), (j % page).to(DEV)
        k, v = k_all[blocks, offs].permute(1, 0, 2)[:, None], v_all[blocks, offs].permute(1, 0, 2)[:, None]   # [H, 1, c, D]
        fine = v.isfinite()
        v, odd = v.masked_fill(~fine, 0.0), [(v == math.inf).double(), (v == -math.inf).double(), v.isnan().double()]
        step = max(1, (1 << 26) // (Hq * c))
        for a in range(0, n, step):
            b = min(n, a + step)
            rows = slice(cu[s] + a, cu[s] + b)
            q = q_all[rows].unflatten(1, (H, -1)).permute(1, 2, 0, 3)                                          # [H, G, b - a, D]
            p = torch.arange(c - n + a, c - n + b, device=DEV)[:, None]
            at_key = torch.arange(c, device=DEV)
            seen = at_key <= p
            if window is not None:
                seen &= (p - at_key < window) | (at_key < sinks)
            score = (q @ k.transpose(-1, -2)) * D ** -0.5
            size = (q.abs() @ k.abs().transpose(-1, -2)) * D ** -0.5
            reach = max(reach, size.masked_fill(~seen, 0.0).nan_to_num(0.0).amax().item())
            keys = max(keys, int(seen.sum(-1).max()))
            w = torch.softmax(score.masked_fill(~seen, -math.inf), -1).masked_fill(~seen.any(-1, keepdim=True), 0.0)
            o = w @ v
            if not fine.all():
                up, down, nan = (seen.double() @ x for x in odd)
                o = o + torch.where(up > 0, math.inf, 0.0) + torch.where(down > 0, -math.inf, 0.0)
                o = torch.where(nan > 0, math.nan, o)
            out[rows] = o.permute(2, 0, 1, 3).flatten(1, 2)
            mass[rows] = (w @ v.abs()).permute(2, 0, 1, 3).flatten(1, 2)
        top = max(top, v.abs().max().item())
    return ref.Attended(out.cpu(), mass.cpu(), reach, keys, top)


def check64(case: Case, **kw) -> torch.Tensor:
    got = case.call(**kw)
    kt.check_device_status(0)
    want = attended64(case, **kw)
    fine, res = want.out.isfinite(), got.cpu().double()
    kind = lambda x: x.masked_fill(fine, 0.0).nan_to_num(7.0, 8.0, 9.0)  # noqa: E731
    wrong = int((kind(res) != kind(want.out)).sum())
    assert wrong == 0, f"{wrong} elements that are not finite differ"
    err, lim = (res - want.out)[fine].abs(), bound(want, case.dtype, case.q4, case.dim)[fine]
    worst = (err / lim.clamp(min=1e-30)).max().item() if err.numel() else 0.0
    assert not err.isnan().any() and (err <= lim).all(), f"worst error is {worst:.3g} of its bound"
    return got


def items_a_cta(q_lens, group, kv_heads):
    """Items per CTA of the kernel for many rows (a persistent CTA per SM), which takes calls of more rows a sequence
    than either crossover."""
    rows = -(-sum(q_lens) // len(q_lens)) * group
    assert rows > 24
    tokens = (128 if rows <= 128 else 256) // group
    return sum(-(-q // tokens) for q in q_lens) * kv_heads / torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(None, 0), (70, 3)])
@pytest.mark.parametrize("q_of", [(0, 1, 5, 31, 32, 33, 64, 65, 130), (1, 2, 9, 17, 32, 33)], ids=["two-tiles", "one-tile"])
def test_many_items_with_keys_on_each_cta(require_gpu, dtype, q4, dim, window, sinks, q_of):
    """Each persistent CTA takes many items in a row: items of one row tile and of two, of one key tile and of several,
    without keys and without tokens in any order; more sequences than a warp has lanes."""
    rng = random.Random(dim + len(q_of))
    q_lens = [rng.choice(q_of) for _ in range(150)]
    ctx = [0 if rng.random() < 0.05 else max(0, q + rng.choice((0, 0, -3, 3, 90, 300))) for q in q_lens]
    case = Case(ctx, 32, 8, dim, 16, dtype, q4, q_lens=q_lens, seed=17)
    assert items_a_cta(q_lens, 4, 8) > 6
    first = check64(case, window=window, sinks=sinks)
    assert torch.equal(first, case.call(window=window, sinks=sinks))


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (1000, 5)])
def test_long_prompts(require_gpu, dtype, q4, window, sinks):
    q_lens = [3001, 700, 1]
    case = Case([3001, 2111, 1500], 16, 4, 128, 64, dtype, q4, q_lens=q_lens, seed=18)
    check64(case, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
def test_chunks_whose_keys_are_split(require_gpu, dtype, q4):
    """Few items and long contexts: the key axis of the kernel for many rows is split too."""
    for dim, group, q_lens, ctx in ((128, 4, [40, 100], [5000, 2900]), (64, 1, [70, 3], [4000, 3])):
        case = Case(ctx, group, 1, dim, 16, dtype, q4, q_lens=q_lens, seed=dim)
        assert -(-sum(q_lens) // 2) * group > 24
        check64(case)
        check64(case, window=2500, sinks=130)


def spoil(case: Case, s: int, j: int, what: float, first: int, last: int, plane="v"):
    """Elements first to last - 1 of key or value j of sequence s, of every kv head, become `what` (in a 4-bit cache
    their groups of 16 become NaN)."""
    blk, off = int(case.tables[s, j // case.page]), j % case.page
    cache = case.k if plane == "k" else case.v
    if not case.q4:
        cache[blk, off, :, first:last] = what
        return
    H, page, dim = cache.shape[2], case.page, case.dim
    scales = cache[blk].view(H, -1)[:, page * dim // 2:].view(H, page, dim // 16)
    scales[:, off, first // 16:-(-last // 16)] = 0x7F


# Decode (single tokens, keys split), drafted tokens (the same kernel), chunks (the kernel for many rows, keys split)
# and prompts (the same, several items a CTA).
SPOILED = [([3000, 2500], None, 4, 1), ([3000, 2500], [4, 3], 4, 1), ([3000, 2500], [70, 90], 4, 1), ([900, 1400], [900, 700], 32, 8)]


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ctx,q_lens,heads,kv_heads", SPOILED, ids=["decode", "draft", "chunk", "prompt"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (300, 5)])
def test_values_that_are_not_finite_in_long_contexts(require_gpu, dtype, q4, dim, ctx, q_lens, heads, kv_heads, window, sinks):
    """Infinities and NaN among the values, some seen by all rows, some by a part of a tile's rows, some of both signs, and
    a NaN key near the end: each element of each row is what the formula gives, and no wait runs out."""
    case = Case(ctx, heads, kv_heads, dim, 16, dtype, q4, q_lens=q_lens, seed=19)
    for s, c in enumerate(ctx):
        n = 1 if q_lens is None else q_lens[s]
        for j, what, first, last in ((1, math.inf, 0, 3), (c // 2, math.nan, 17, 18), (c - n // 2 - 1, math.inf, 32, 40),
                                     (c - n // 3 - 1, -math.inf, 36, 44), (c - 2, math.nan, 50, 51),
                                     (max(0, c - n - 290), math.nan, 60, 61), (c - n // 4 - 1, -math.inf, 0, 64)):
            spoil(case, s, j, what, first, last)
    check64(case, window=window, sinks=sinks)
    spoil(case, 1, ctx[1] - 2, math.nan, 5, 6, "k")
    check64(case, window=window, sinks=sinks)


@pytest.mark.parametrize("q4", [False, True])
def test_a_value_that_is_not_finite_costs_little(require_gpu, q4):
    """One such value that most rows rightly see takes milliseconds, not seconds (0.16 ms without it, 0.4 to 1.0 with);
    one at the end, for which 244 rows of four items have to be computed again, 93."""
    def milliseconds(case):
        f = at.paged_attention_q4 if q4 else at.paged_attention
        args = case.q.to(DEV), case.k, case.v, case.tables.to(DEV), case.ctx.to(DEV), 16
        cu = case.cu.to(DEV)
        best = math.inf
        for _ in range(3):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            f(*args, cu_seqlens_q=cu)
            end.record()
            end.synchronize()
            best = min(best, start.elapsed_time(end))
        kt.check_device_status(0)
        return best

    for ctx, q_lens in (([4096], [4096]), ([20000], [5])):
        for j, most in ((3, 30), (ctx[0] // 2, 30), (ctx[0] - 3, 500)):      # the last: rows of its own tile do not see it
            case = Case(ctx, 16, 4, 128, 16, torch.float16, q4, q_lens=q_lens, seed=21)
            milliseconds(case)
            spoil(case, 0, j, math.nan, 9, 10)
            assert milliseconds(case) < most


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
@pytest.mark.parametrize("tokens,copies", [(1, 1200), (3, 1200), (40, 75), (3, 1)], ids=["decode", "draft", "chunk", "split"])
def test_a_long_tail_behind_strong_sinks_counts(require_gpu, dtype, q4, tokens, copies):
    """131070 keys, eight strong ones at the start (one for each part of a tile that has a maximum of its own) and a tail of
    about 2^-26 of their weight each, together 2^-12, whose values alone are not 0. A weight in fp16 is off by at most 2^-25
    of 2^7 times the largest, so the last term of the bound is n 2^-32 max |v| here. The same sequence many times over
    leaves the keys of an item in one piece."""
    n, dim, page, heads = 131070, 64, 256, 2
    case = Case([n], 4 * heads, heads, dim, page, dtype, q4, q_lens=[tokens], seed=22)
    g = torch.Generator().manual_seed(23)
    k, v = torch.zeros(n, heads, dim), 1 + 0.125 * torch.randn(n, heads, dim, generator=g).clamp(-3, 3)
    k[:, :, 16:32] = 0.25 * torch.randn(n, heads, 16, generator=g)
    for j in range(0, 128, 16):
        k[j], v[j] = 0.0, 0.0
        k[j, :, 0] = 6.0                                            # on the grid of a 4-bit row
    slots = case.tables[0].long()[torch.arange(n) // page] * page + torch.arange(n) % page
    (at.store_kvcache_q4 if q4 else at.store_kvcache)(k.to(dtype).to(DEV), v.to(dtype).to(DEV), case.k, case.v, slots.to(DEV), page)
    case.q = 0.5 * torch.randn(case.q.shape, generator=g)
    case.q[:, :, 0] = 26 * math.log(2) / 6 * dim ** 0.5
    case.q = case.q.to(dtype)
    want = attended64(case)
    f = at.paged_attention_q4 if q4 else at.paged_attention
    got = f(case.q.repeat(copies, 1, 1).to(DEV), case.k, case.v, case.tables.repeat(copies, 1).to(DEV),
            case.ctx.repeat(copies).to(DEV), page,
            cu_seqlens_q=None if tokens == 1 else torch.arange(copies + 1, dtype=torch.int32, device=DEV) * tokens)
    kt.check_device_status(0)
    assert torch.equal(got, got[:tokens].repeat(copies, 1, 1))
    half = q4 or dtype == torch.float16
    lim = bound(want, dtype, q4, dim) - want.keys * 2.0 ** -25 * want.top + (want.keys * 2.0 ** -32 * want.top if half else 0.0)
    assert 2.0 ** -13 < want.out.min() and want.out.max() < 2.0 ** -11 and lim.max() < 2.0 ** -13
    err = (got[:tokens].cpu().double() - want.out).abs()
    assert (err <= lim).all(), f"worst error is {(err / lim).max():.3g} of its bound"


@pytest.mark.parametrize("q_lens", [None, [3, 2], [40, 30]], ids=["decode", "draft", "chunk"])
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_beyond_fp32_are_infinite(require_gpu, dim, q_lens):
    """Products that fit into fp32 until they are scaled: NaN for the rows that see one, the others as ever."""
    case = Case([90, 70], 4, 1, dim, 16, torch.bfloat16, False, q_lens=q_lens, seed=24)
    case.q[:, 0] *= 2.0 ** 50                                       # one head of four
    case.k *= 2.0 ** 65
    got = case.call(scale=2.0 ** 14)
    kt.check_device_status(0)
    assert got[:, 0].isnan().all() and got[:, 1:].isfinite().all() and got[:, 1:].abs().amax(-1).gt(0).all()


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
@pytest.mark.parametrize("ctx,q_lens", [([300, 200], None), ([300, 200], [3, 2]), ([300, 200], [40, 30]), ([4000], [60])],
                         ids=["decode", "draft", "chunk", "split"])
def test_scores_far_apart_leave_the_key_of_the_largest(require_gpu, dtype, q4, ctx, q_lens):
    """Scores of 2^26 and more: their roundings are far larger than 1, and what is left of a row is the value of its best key."""
    dim = 64
    case = Case(ctx, 4, 1, dim, 16, dtype, q4, q_lens=q_lens, seed=25)
    size = 2.0 ** 13 if dtype == torch.float16 else 2.0 ** 25
    case.q = (case.q.float().clamp(-4, 4) * size).to(dtype)
    if not q4:
        case.k = (case.k.float().clamp(-4, 4) * 2.0 ** 13).to(dtype)
    k, v = case.values()
    got = case.call().cpu().double()
    kt.check_device_status(0)
    cu = case.cu.tolist() if case.cu is not None else range(len(ctx) + 1)
    clear = 0
    for s, c in enumerate(ctx):
        j = torch.arange(c)
        ids = case.tables[s].long()[j // 16]
        keys, values = k[ids, j % 16, 0], v[ids, j % 16, 0]
        for t in range(cu[s], cu[s + 1]):
            p = c - cu[s + 1] + t
            q = case.q[t].double()
            score, reach = q @ keys[:p + 1].T * dim ** -0.5, (q.abs() @ keys[:p + 1].abs().T * dim ** -0.5).amax()
            (first, second), best = score.topk(2, -1).values.unbind(-1), score.argmax(-1)
            # each score is off by (D + 8) half steps of fp32 at most; other keys' weights stay below 2^-40
            sure = first - second > 2 * (dim + 8) * 2.0 ** -24 * reach + 40
            clear += int(sure.sum())
            err = (got[t] - values[best]).abs()
            # half a step of the output, and half a step of the best key's weight, which is rounded for the products (it is
            # 2^x, x the rounding of score * scale) but not in their sum: w (1 + d) v / w
            step = HALF_STEP[dtype] + (2.0 ** -11 if q4 else HALF_STEP[dtype])
            assert (err <= step * (1 + 2.0 ** -8) * values[best].abs() + 2.0 ** -30 * values.abs().max())[sure].all()
    assert clear > (4 if q_lens is None else 2 * sum(q_lens))


@pytest.mark.parametrize("q4", [False, True])
def test_a_single_token_or_head_may_have_any_stride(require_gpu, q4):
    """The stride of a dimension of one entry of the query, of `out` and of the rows to store means nothing."""
    f = at.paged_attention_q4 if q4 else at.paged_attention
    for heads, tokens in ((4, 1), (1, 1), (1, 3)):
        case = Case([70], heads, 1, 64, 16, torch.bfloat16, q4, q_lens=[tokens], seed=27)
        want = case.check()
        strides = (257 if tokens == 1 else heads * 64, 3 if heads == 1 else 64, 1)
        memory = torch.zeros(2, 2048, dtype=torch.bfloat16, device=DEV)
        q, out = (m.as_strided(case.q.shape, strides) for m in memory)
        q.copy_(case.q)
        got = f(q, case.k, case.v, case.tables.to(DEV), case.ctx.to(DEV), 16, cu_seqlens_q=case.cu.to(DEV), out=out)
        assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)
        odd = torch.zeros(2049, dtype=torch.bfloat16, device=DEV)[1:].as_strided(case.q.shape, strides)
        odd.copy_(case.q)
        assert torch.equal(f(odd, case.k, case.v, case.tables.to(DEV), case.ctx.to(DEV), 16, cu_seqlens_q=case.cu.to(DEV)), want)
    x = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(28)).to(torch.bfloat16)
    caches = [torch.zeros(1, 16, 2, at.q4_row_bytes(64), dtype=torch.uint8, device=DEV) for _ in range(4)]
    slot = torch.tensor([3], device=DEV)
    at.store_kvcache_q4(x.to(DEV), x.to(DEV), caches[0], caches[1], slot, 16)
    odd = torch.zeros(2, 512, dtype=torch.bfloat16, device=DEV).as_strided((2, 1, 2, 64), (512, 131, 64, 1))
    odd.copy_(x.expand(2, 1, 2, 64))
    at.store_kvcache_q4(odd[0], odd[1], caches[2], caches[3], slot, 16)
    assert int(caches[0].sum()) > 0 and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


@pytest.mark.parametrize("dtype,q4", TYPES, ids=IDS)
@pytest.mark.parametrize("tokens", [1, 3, 40], ids=["decode", "draft", "chunk"])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_late_key_eight_binades_above_a_large_score(require_gpu, dtype, q4, tokens, dim):
    """The largest weight that a maximum is not renewed for, at scores whose neighbours are 4 to 8 apart: 2^8 times the
    first key's, still finite in the products. Scores are exact here (in units of log2, with scale = ln 2)."""
    n, page = 200, 16
    case = Case([n], 4, 1, dim, page, dtype, q4, q_lens=[tokens], seed=30)
    high = 1536.0 if q4 else 2.0 ** 13
    k, v = torch.zeros(n, 1, dim), torch.zeros(n, 1, dim)
    k[0, 0, 0] = k[128, 0, 0] = high
    k[128, 0, 16], k[128, 0, 17] = 8.0, 12.0                        # 12 gives the group the scale 2; no query reads it
    v[0], v[128] = 6.0, 3.0
    slots = case.tables[0].long()[torch.arange(n) // page] * page + torch.arange(n) % page
    (at.store_kvcache_q4 if q4 else at.store_kvcache)(k.to(dtype).to(DEV), v.to(dtype).to(DEV), case.k, case.v, slots.to(DEV), page)
    case.q = torch.zeros_like(case.q)
    case.q[:, :, 0] = 2.0 ** 13 if not q4 else 2.0 ** 16 if dtype == torch.bfloat16 else 2.0 ** 15
    case.q[:, :, 16] = 1.0
    got = case.call(scale=math.log(2)).cpu().double()
    kt.check_device_status(0)
    want = (6.0 + 256 * 3.0) / 257
    # half a step of the output, of each weight and, twice, the exponentials' 2^-18
    step = HALF_STEP[dtype] + (2.0 ** -11 if q4 else HALF_STEP[dtype]) + 2.0 ** -17
    assert ((got - want).abs() <= step * want).all()


# ----------------------------------------------------------------------------------------------
# Refusals
# ----------------------------------------------------------------------------------------------

def test_refusals(require_gpu):
    case = Case([20, 30], 4, 2, 64, 16, torch.float16, False, seed=1)
    q, k, v, table, ctx = case.q.to(DEV), case.k, case.v, case.tables.to(DEV), case.ctx.to(DEV)

    def call(q=q, k=k, v=v, table=table, ctx=ctx, bs=16, **kw):
        return at.paged_attention(q, k, v, table, ctx, bs, **kw)

    with pytest.raises(TypeError):
        call(q=q.float())
    with pytest.raises(TypeError):
        call(q=q.bfloat16())
    with pytest.raises(TypeError):
        call(table=table.long())
    with pytest.raises(TypeError):
        call(ctx=ctx.long())
    with pytest.raises(TypeError):
        call(cu_seqlens_q=torch.tensor([0, 1, 2], device=DEV))
    with pytest.raises(RuntimeError, match="num_seqs"):
        call(cu_seqlens_q=torch.tensor([0, 2], dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="one token"):
        call(q=q[:1])
    with pytest.raises(RuntimeError, match="multiple"):
        call(q=q[:, :3])
    with pytest.raises(RuntimeError, match="head_dim"):
        call(q=q[..., :32])
    with pytest.raises(RuntimeError):
        call(bs=32)
    with pytest.raises(RuntimeError, match="strides"):
        call(v=v.transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(ValueError):
        call(window=0, sinks=3)
    with pytest.raises(ValueError):
        call(window=-1)
    with pytest.raises(RuntimeError, match="scale"):
        call(scale=0.0)
    with pytest.raises(RuntimeError, match="scale"):
        call(scale=float("nan"))
    with pytest.raises(RuntimeError):
        call(out=torch.empty(2, 4, 64, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(RuntimeError, match="out must not"):
        call(out=q)
    with pytest.raises(RuntimeError, match="CUDA"):
        call(q=q.cpu(), k=k.cpu(), v=v.cpu(), table=table.cpu(), ctx=ctx.cpu())
    with pytest.raises(RuntimeError):
        call(table=table.cpu())
    with pytest.raises(TypeError):
        at.paged_attention_q4(q, k, v, table, ctx, 16)
    row = at.q4_row_bytes(64)
    kc = torch.zeros(4, 16, 2, row, dtype=torch.uint8, device=DEV)
    with pytest.raises(RuntimeError, match="4-bit cache"):
        at.paged_attention_q4(q, kc[..., :32], kc[..., :32], table, ctx, 16)
    with pytest.raises(RuntimeError, match="contiguous"):
        at.paged_attention_q4(q, kc[:, :, ::2].expand(4, 16, 2, row), kc[:, :, ::2].expand(4, 16, 2, row), table, ctx, 16)
    with pytest.raises(RuntimeError, match="power"):
        at.paged_attention_q4(q, kc, kc.clone(), table, ctx, 16, k_scale=3.0)
    small = torch.zeros(4, 8, 2, row, dtype=torch.uint8, device=DEV)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        at.paged_attention_q4(q, small, small.clone(), table, ctx, 8)
    x = torch.zeros(3, 2, 64, dtype=torch.float16, device=DEV)
    slots = torch.arange(3, device=DEV)
    with pytest.raises(TypeError):
        at.store_kvcache_q4(x.float(), x.float(), kc, kc.clone(), slots, 16)
    with pytest.raises(TypeError):
        at.store_kvcache_q4(x, x, kc, kc.clone(), slots.int(), 16)
    with pytest.raises(AssertionError):
        at.store_kvcache_q4(x, x, kc, kc.clone(), slots[:2], 16)
    with pytest.raises(RuntimeError):
        at.store_kvcache_q4(x[:, :1], x[:, :1], kc, kc.clone(), slots, 16)
    with pytest.raises(RuntimeError, match="power"):
        at.store_kvcache_q4(x, x, kc, kc.clone(), slots, 16, v_scale=0.0)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        at.store_kvcache_q4(x, x, small, small.clone(), slots, 8)
    with pytest.raises(TypeError):
        at.load_kvcache_q4(kc, kc, slots, 16, dtype=torch.float32)
    torch.cuda.synchronize()
    kt.check_device_status(0)


@pytest.mark.gpu
def test_an_output_whose_rows_share_memory_is_refused(require_gpu):
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device=DEV)
    tables = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    ctx = torch.ones(2, dtype=torch.int32, device=DEV)
    for out in (torch.empty(1, 4, 64, dtype=torch.bfloat16, device=DEV).expand(2, 4, 64),
                torch.empty(2, 1, 64, dtype=torch.bfloat16, device=DEV).expand(2, 4, 64)):
        with pytest.raises(RuntimeError, match="must not overlap"):
            at.paged_attention(q, cache, cache.clone(), tables, ctx, 16, out=out)


def test_an_output_whose_tokens_and_heads_share_rows_is_refused(require_gpu):
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device=DEV)
    tables = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    ctx = torch.ones(2, dtype=torch.int32, device=DEV)
    memory = torch.empty(4096, dtype=torch.bfloat16, device=DEV)
    for strides in ((64, 64, 1), (128, 64, 1), (64, 96, 1), (128, 128, 1)):
        with pytest.raises(RuntimeError, match="must not overlap"):
            at.paged_attention(q, cache, cache.clone(), tables, ctx, 16, out=memory.as_strided(q.shape, strides))
    for strides in ((64, 128, 1), (256, 64, 1), (192, 128, 1)):
        got = at.paged_attention(q, cache, cache.clone(), tables, ctx, 16, out=memory.as_strided(q.shape, strides))
        assert got.eq(0).all()


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("heads", [1, 20])
def test_offsets_out_of_order_are_flagged_wherever_they_stand(require_gpu, q4, heads):
    """Also where the search for a sequence passes over the one whose end is before its start (heads: either kernel)."""
    good = [0, 1, 2, 4, 6, 8, 12, 16]
    case = Case([20] * 7, heads, 1, 64, 16, torch.float16, q4, q_lens=[b - a for a, b in zip(good, good[1:])], seed=29)
    case.call()
    kt.check_device_status(0)
    for i, bad in ((2, 9), (1, 13), (6, 3), (3, 17), (5, -1), (7, 11), (0, 2)):
        cu = list(good)
        cu[i] = bad
        case.cu = torch.tensor(cu, dtype=torch.int32)
        case.call()
        with pytest.raises(_capi.KvxError, match="length"):
            kt.check_device_status(0)
