"""The paged fp8 cache on the GPU against the oracle in 64 bits.

Bits are compared where rounding is to the nearest of exactly known numbers: the cache after an append, what is read
back.  Attention: K and V enter exactly, scores and sums are fp32 (relative errors of 2^-20 at the lengths here), a
probability is rounded to fp16 at most once (half a step, 2^-11, relative to itself: A = softmax . |V| bounds what that
can move) and O once to its own type.  So |O - ref| <= eps/2 |ref| + 1.25 * 2^-11 A, the quarter for the fp32 part and for
probabilities below fp16's normal range, and half of fp16's smallest number for outputs below its own.  The log-sum-exp: scores of size s carry
errors of 2^-20 s."""
import math

import pytest
import torch

from cutlass_flash_atten_fp8_b200 import (PagedKVCache, _lib, api, check_status, flash_attention_paged_kv, flash_attention_v2_cutlass,
                                          paged_kv_append, paged_kv_read)
from oracle import paged_kv_oracle as po

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def bits(t):
    return t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()]).cpu()


def filled(heads, D, P, dtype, seqs, seed, spare=3):
    """A pool on the host whose pages hold values of very different size, a table with wild numbers behind each
    sequence's pages, and NaN wherever nothing of a sequence is held."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-s // P) for _, s in seqs]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(seqs), max(need) + 2), 2 ** 31 - 1, dtype=torch.int32)
    table[:, -1] = -7
    cache = [torch.randn(pages, heads, P, D, generator=g).mul_(40).to(dtype) for _ in range(2)]
    cache += [torch.exp2(torch.randint(-9, -3, (pages, heads), generator=g).float()) for _ in range(2)]
    used = torch.zeros(pages, P, dtype=torch.bool)
    at = 0
    for b, (_, s) in enumerate(seqs):
        for p in range(need[b]):
            table[b, p] = order[at]
            used[order[at], :min(P, s - p * P)] = True
            at += 1
    for x8 in cache[:2]:
        x8.copy_(torch.where(used[:, None, :, None], x8.float(), torch.nan).to(dtype))
    for d in cache[2:]:
        d[~used.any(1)] = torch.nan
    return cache, table


def ranges(seqs, lead=0, tail=0):
    """cu_seqlens (None if even and nothing around), rows, seqlens."""
    n = [x for x, _ in seqs]
    cu = torch.tensor([lead] + n).cumsum(0).to(torch.int32)
    even = len(set(n)) == 1 and not lead and not tail
    return (None if even else cu), int(cu[-1]) + tail, torch.tensor([s for _, s in seqs], dtype=torch.int32)


def to(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


def rows(T, heads, D, dtype, seed, fused, cu, seqs):
    """[T, heads, D] on the GPU, part of a wider tensor if fused; NaN in rows of no sequence."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, heads + (3 if fused else 0), D, generator=g).to(dtype)
    if cu is not None:
        x[:int(cu[0])] = math.nan
        x[int(cu[-1]):] = math.nan
    x = x.to(DEV)
    return x[:, 1:1 + heads] if fused else x


# new tokens and length (with them) of each sequence
APPENDS = {
    "one token": [(1, 1)], "one token, page begins": [(1, 17)], "one token, page ends": [(1, 16)], "mid page": [(1, 9), (1, 300), (1, 33)],
    "nothing new": [(0, 5), (3, 3), (0, 0), (2, 31)], "across pages": [(40, 47), (129, 260), (17, 32), (2, 129)], "prompts": [(300, 300), (1, 1), (77, 77), (128, 128)],
}
SHAPES = [(1, 32, 16), (2, 64, 16), (3, 96, 32), (2, 128, 64), (1, 256, 128), (2, 224, 16)]


@pytest.mark.parametrize("name", APPENDS)
@pytest.mark.parametrize("heads,D,P", SHAPES)
@pytest.mark.parametrize("half,fp8", [(torch.float16, E4M3), (torch.bfloat16, E4M3), (torch.bfloat16, E5M2), (torch.float16, E5M2)])
def test_append(name, heads, D, P, half, fp8):
    seqs = APPENDS[name]
    lead, tail = (2, 3) if name == "nothing new" else (0, 0)
    cu, T, lens = ranges(seqs, lead, tail)
    cache, table = filled(heads, D, P, fp8, seqs, seed=1 + D)
    k, v = (rows(T, heads, D, half, s, name == "across pages", cu, seqs) for s in (2, 3))
    k *= 37.0                                                     # K outgrows the older scales, V mostly does not
    k[lead, 0, 0] = 0.0
    v[lead, 0, 0], v[lead, 0, 1] = math.inf, math.nan
    want = po.append(cache, k.cpu(), v.cpu(), table, lens, cu)
    got = PagedKVCache(*to(DEV, *cache))
    paged_kv_append(got, k, v, *to(DEV, table, lens), cu_seqlens=None if cu is None else cu.to(DEV))
    check_status(DEV)
    for w, g in zip(want[2:], got[2:]):
        assert torch.equal(bits(w), bits(g))
    for w, g in zip(want[:2], got[:2]):
        g = g.cpu()
        nan = torch.isnan(w.float())
        assert torch.equal(nan, torch.isnan(g.float()))           # a NaN's sign is nobody's
        assert torch.equal(bits(w)[~nan], bits(g)[~nan])


@pytest.mark.parametrize("half", [torch.float16, torch.bfloat16])
def test_append_of_nothing_but_zeros_and_of_the_extremes(half):
    """Zeros take the smallest scale and do not spoil the page for what follows; the largest and smallest numbers clamp."""
    P, D = 16, 64
    cache, table = filled(1, D, P, E4M3, [(4, 4)], seed=3)
    got = PagedKVCache(*to(DEV, *cache))
    host = cache
    info = torch.finfo(half)
    for i, value in enumerate((0.0, info.tiny, 1e-3, info.max)):
        x = torch.full((1, 1, D), value, dtype=half)
        s = torch.tensor([i + 1], dtype=torch.int32)
        host = po.append(host, x, -x, table, s)
        paged_kv_append(got, x.to(DEV), -x.to(DEV), *to(DEV, table, s))
        check_status(DEV)
        for w, g in zip(host[2:], got[2:]):
            assert torch.equal(bits(w), bits(g))
        page = int(table[0, 0])
        for w, g in zip(host[:2], got[:2]):
            assert torch.equal(w[page, :, :i + 1].float(), g.cpu()[page, :, :i + 1].float())


@pytest.mark.parametrize("name", APPENDS)
@pytest.mark.parametrize("heads,D,P", SHAPES)
@pytest.mark.parametrize("half,fp8", [(torch.float16, E4M3), (torch.bfloat16, E4M3), (torch.bfloat16, E5M2)])
def test_read(name, heads, D, P, half, fp8):
    seqs = APPENDS[name]
    cu, T, lens = ranges(seqs, *((2, 3) if name == "nothing new" else (0, 0)))
    cache, table = filled(heads, D, P, fp8, seqs, seed=1 + D)
    got = paged_kv_read(to(DEV, *cache), *to(DEV, table, lens), T, cu_seqlens=None if cu is None else cu.to(DEV), dtype=half)
    check_status(DEV)
    mine = slice(None) if cu is None else slice(int(cu[0]), int(cu[-1]))
    for w, g in zip(po.read(cache, table, lens, T, cu), got):
        assert g.shape == (T, heads, D)
        assert torch.equal(bits(w[mine].to(half)), bits(g[mine]))


def check_attention(q, cache, table, lens, causal, scale, cu, out, lse):
    want, want_lse, A = po.attention(q.cpu(), cache, table, lens, causal, scale, cu)
    held = ~torch.isnan(want)
    got, lse = out.double().cpu(), lse.double().cpu()
    assert torch.equal(torch.isnan(got) & held, torch.zeros_like(held))
    half_step = torch.finfo(q.dtype).eps / 2
    limit = half_step * want.abs() + 1.25 * 2.0 ** -11 * A + 2.0 ** -25
    off = ((got - want).abs() - limit)[held]
    assert off.numel() == 0 or float(off.max()) <= 0, float(((got - want).abs() / limit)[held].max())
    rows_held = held[:, :, 0]
    a, b = lse[rows_held], want_lse[rows_held]
    assert torch.equal(a == -math.inf, b == -math.inf)
    fin = b > -math.inf
    assert bool(((a - b).abs()[fin] <= 2.0 ** -20 * (b.abs()[fin] + 16)).all())
    return held


def attend(seqs, H, Hk, D, P, half, fp8, causal, seed=0, fused=False, lead=0, tail=0, scale=None):
    cu, T, lens = ranges(seqs, lead, tail)
    cache, table = filled(Hk, D, P, fp8, seqs, seed=seed + D)
    q = rows(T, H, D, half, seed + 5, fused, cu, seqs)
    scale = 2.0 / math.sqrt(D) if scale is None else scale
    guard = torch.full((T * H * D + 64,), math.nan, dtype=half, device=DEV)
    out, lse = flash_attention_paged_kv(q, to(DEV, *cache), *to(DEV, table, lens), causal, scale,
                                        cu_seqlens=None if cu is None else cu.to(DEV), out=guard[:T * H * D].view(T, H, D), return_lse=True)
    check_status(DEV)
    assert bool(torch.isnan(guard[T * H * D:]).all())
    held = check_attention(q, cache, table, lens, causal, scale, cu, out, lse)
    assert bool(torch.isnan(out.cpu()[~held]).all())              # rows of no sequence are left as they were
    return out


TOKENS = {"one key": [(1, 1)], "short": [(1, 15), (1, 16), (1, 17)], "tile ends": [(1, 31), (1, 32), (1, 33), (1, 63), (1, 64), (1, 65)],
          "long and short": [(1, 3000), (1, 2), (1, 513)], "many": [(1, 7 * i + 1) for i in range(70)]}


@pytest.mark.parametrize("name", TOKENS)
@pytest.mark.parametrize("H,Hk,D,P", [(1, 1, 32, 16), (4, 2, 64, 16), (8, 1, 128, 32), (9, 3, 96, 64), (5, 1, 256, 128), (16, 1, 128, 16),
                                      (32, 2, 64, 64), (17, 1, 160, 16), (6, 6, 128, 128)])
@pytest.mark.parametrize("half,fp8", [(torch.float16, E4M3), (torch.bfloat16, E5M2)])
def test_attention_of_single_tokens(name, H, Hk, D, P, half, fp8):
    attend(TOKENS[name], H, Hk, D, P, half, fp8, True)


SEVERAL = {"two": [(2, 2), (2, 40)], "drafts": [(4, 100), (3, 3), (5, 700), (1, 64)], "more than there are": [(6, 3), (2, 0), (1, 1)],
           "nothing new": [(0, 50), (3, 60), (0, 0)], "mixed": [(150, 150), (1, 400), (130, 1000), (1, 1), (7, 64)], "prompts": [(257, 257), (128, 128), (64, 64)],
           "chunk": [(200, 900)]}


@pytest.mark.parametrize("name", SEVERAL)
@pytest.mark.parametrize("H,Hk,D,P", [(2, 2, 64, 16), (4, 1, 128, 16), (6, 2, 96, 32), (8, 2, 128, 64), (2, 1, 256, 64), (5, 1, 128, 128), (3, 3, 32, 32)])
@pytest.mark.parametrize("half,fp8,causal", [(torch.float16, E4M3, True), (torch.bfloat16, E4M3, False), (torch.bfloat16, E5M2, True), (torch.float16, E5M2, False)])
def test_attention_of_several_tokens(name, H, Hk, D, P, half, fp8, causal):
    around = (3, 5) if name in ("nothing new", "drafts") else (0, 0)
    attend(SEVERAL[name], H, Hk, D, P, half, fp8, causal, seed=7, fused=name in ("mixed", "two"), lead=around[0], tail=around[1])


@pytest.mark.parametrize("seqs", [[(1, 700), (1, 90)], [(140, 500)]], ids=["tokens", "chunk"])
@pytest.mark.parametrize("half", [torch.float16, torch.bfloat16])
def test_attention_with_scales_of_very_different_size(seqs, half):
    """Pages whose scales span fifty binades, steep softmaxes, and a query row far from 1."""
    H, Hk, D, P = 4, 2, 64, 16
    cu, T, lens = ranges(seqs)
    cache, table = filled(Hk, D, P, E4M3, seqs, seed=11)
    g = torch.Generator().manual_seed(12)
    pages = cache[2].shape[0]
    cache[2] = torch.exp2(torch.randint(-30, -3, (pages, Hk), generator=g).float())
    cache[3] = torch.exp2(torch.randint(-40, 11, (pages, Hk), generator=g).float())
    q = rows(T, H, D, half, 13, False, cu, seqs)
    q[0] *= 2.0 ** 8
    if half is torch.bfloat16:
        q[0, 1] *= 2.0 ** 20                                      # beyond fp16
        cache[2][:] *= 2.0 ** -18
    q, scale = q, 1.0
    dev = to(DEV, *cache)
    out, lse = flash_attention_paged_kv(q, dev, *to(DEV, table, lens), True, scale, return_lse=True)
    check_status(DEV)
    want, want_lse, A = po.attention(q.cpu(), cache, table, lens, True, scale, cu)
    fits = want.abs() < torch.finfo(half).max
    # scores reach 2^12 here: fp32 sums carry them to 2^-24 of sum |q k|, and a probability moves by as much
    k = [po.keys_values(cache, table, b, s)[0] for b, (_, s) in enumerate(seqs)]
    qd = q.cpu().double()
    worst = max(float(torch.einsum("ihd,jhd->hij", qd[f:f + n].abs(), k[b].repeat_interleave(H // Hk, 1).abs()).max()) for b, f, n, _ in po.spans(lens, cu, T))
    p_err = math.expm1(worst * 2.0 ** -22)
    limit = torch.finfo(half).eps / 2 * want.abs() + (1.25 * 2.0 ** -11 + p_err) * A + 2.0 ** -25
    # a probability below fp16's normal range is rounded relative to the largest contribution, 448 * 2^-25 of it
    limit = limit + 448 * 2.0 ** -25 * A.amax(-1, keepdim=True)
    assert bool(((out.double().cpu() - want).abs() <= limit)[fits].all())
    assert bool(((lse.double().cpu() - want_lse).abs() <= 2.0 ** -20 * (want_lse.abs() + 16) + worst * 2.0 ** -22).all())


def test_nan_and_infinity_in_held_keys_come_through():
    seqs = [(1, 40), (1, 40)]
    cache, table = filled(1, 64, 16, E4M3, seqs, seed=4)
    cache[1][int(table[0, 1]), 0, 3, 5] = math.nan
    q = rows(2, 2, 64, torch.float16, 5, False, None, seqs)
    out = flash_attention_paged_kv(q, to(DEV, *cache), table.to(DEV), torch.tensor([40, 40], dtype=torch.int32, device=DEV), True, 0.1)[0].cpu()
    check_status(DEV)
    nan = torch.isnan(out)
    assert bool(nan[0, :, 5].all()) and int(nan.sum()) == 2       # column 5 of that sequence alone


GROUPS = [(160, 1, 64), (48, 1, 128), (7, 1, 128), (128, 1, 32), (129, 1, 64), (100, 2, 256)]


@pytest.mark.parametrize("H,Hk,D", GROUPS)
@pytest.mark.parametrize("seqs", [[(1, 300), (1, 40)], [(3, 70), (2, 2), (5, 260)], [(70, 90), (1, 200), (33, 33)]], ids=["tokens", "drafts", "prompts"])
def test_attention_with_groups_of_any_size(H, Hk, D, seqs):
    """Query heads of a K/V head that fill no block of rows, or more than one."""
    attend(seqs, H, Hk, D, 32, torch.bfloat16, E4M3, True, seed=21)


RAGGED = {"forty": [(i % 4, i % 4 + 9 * i % 130) for i in range(40)], "a thousand": [(i % 3, i % 3 + 5 * i % 40) for i in range(1100)],
          "forty prompts": [(33 + 11 * i % 60, 33 + 11 * i % 60 + 7 * (i % 5)) for i in range(40)],
          "one prompt among tokens": [(1, 1 + i % 50) if i != 20 else (900, 900) for i in range(45)]}


@pytest.mark.parametrize("name", RAGGED)
@pytest.mark.parametrize("D,P", [(64, 16), (128, 64)])
def test_attention_of_many_sequences(name, D, P):
    attend(RAGGED[name], 4, 2, D, P, torch.float16, E4M3, True, seed=22, lead=2, tail=1)


@pytest.mark.parametrize("name", ["forty", "a thousand", "forty prompts"])
def test_append_and_read_of_many_sequences(name):
    seqs, heads, D, P, half = RAGGED[name], 2, 64, 16, torch.bfloat16
    cu, T, lens = ranges(seqs, 2, 3)
    cache, table = filled(heads, D, P, E4M3, seqs, seed=23)
    k, v = (rows(T, heads, D, half, s, False, cu, seqs) for s in (24, 25))
    dev, where = PagedKVCache(*to(DEV, *cache)), to(DEV, table, lens)
    paged_kv_append(dev, k, v, *where, cu_seqlens=cu.to(DEV))
    got = paged_kv_read(dev, *where, T, cu_seqlens=cu.to(DEV), dtype=half)
    check_status(DEV)
    after = po.append(cache, k.cpu(), v.cpu(), table, lens, cu)
    for x, y in zip(dev, after):
        assert torch.equal(x.cpu().float().nan_to_num(-1.0), y.float().nan_to_num(-1.0))
    for x, y in zip(got, po.read(after, table, lens, T, cu)):
        assert torch.equal(x[int(cu[0]):int(cu[-1])].cpu().double(), y[int(cu[0]):int(cu[-1])].to(half).double())


@pytest.mark.parametrize("seqs,H,Hk,D,P", [([(130, 3000)], 1, 1, 64, 64), ([(130, 3000)], 4, 2, 128, 16), ([(257, 2600)], 2, 1, 256, 128),
                                            ([(70, 70), (150, 2900)], 2, 1, 128, 32), ([(600, 600)] * 5, 16, 16, 64, 64), ([(300, 333), (0, 3), (700, 700)], 16, 8, 128, 16)],
                         ids=["parts 64", "parts 128", "parts 256", "parts of which some are empty", "more items than SMs", "ragged"])
@pytest.mark.parametrize("half,fp8,causal", [(torch.float16, E4M3, True), (torch.bfloat16, E5M2, False)])
def test_attention_of_prompts_in_parts_and_in_many_items(seqs, H, Hk, D, P, half, fp8, causal):
    """Few items, whose keys are cut into parts and joined; many, which CTAs take over from one another."""
    attend(seqs, H, Hk, D, P, half, fp8, causal, seed=26)


@pytest.mark.parametrize("n_seqs,Hk,length", [(1, 1, 6000), (1, 2, 1500), (12, 2, 900), (20, 2, 700), (2, 4, 100), (30, 4, 1000)])
@pytest.mark.parametrize("H,D", [(1, 64), (4, 128), (9, 256), (8, 32)])
def test_attention_of_single_tokens_by_clusters(n_seqs, Hk, length, H, D):
    """Items few and short enough for a cluster of one to eight CTAs each (and some for which they are not)."""
    attend([(1, max(0, length - 37 * b)) for b in range(n_seqs)], H * Hk, Hk, D, 64, torch.float16, E4M3, True, seed=27)


@pytest.mark.parametrize("seqs", [[(1, 300), (1, 40)], [(4, 300), (4, 40)], [(150, 300), (150, 150)]], ids=["tokens", "drafts", "prompts"])
@pytest.mark.parametrize("D,fp8", [(64, E4M3), (128, E5M2), (256, E4M3)])
def test_scales_of_zero(seqs, D, fp8):
    """A page of scale zero holds zeros: keys that count, with scores of 0, and values that add nothing."""
    H, Hk, P, half = 4, 2, 16, torch.float16
    cu, T, lens = ranges(seqs)
    cache, table = filled(Hk, D, P, fp8, seqs, seed=28)
    cache[2][table[0, 0]] = 0.0
    cache[2][table[0, 2]] = 0.0
    cache[3][table[0, 1]] = 0.0
    cache[3][table[1, 0]] = 0.0
    cache[2][table[1, 1]] = cache[3][table[1, 1]] = 0.0
    q = rows(T, H, D, half, 29, False, cu, seqs)
    out, lse = flash_attention_paged_kv(q, to(DEV, *cache), *to(DEV, table, lens), True, 0.2, return_lse=True)
    check_status(DEV)
    check_attention(q, cache, table, lens, True, 0.2, cu, out, lse)


@pytest.mark.parametrize("seqs", [[(3, 40), (4, 300)], [(40, 200), (5, 5)], [(150, 500), (300, 300), (129, 140)], [(260, 3000)]], ids=["drafts", "pieces", "prompts", "parts"])
@pytest.mark.parametrize("H,Hk,D,P", [(2, 2, 64, 16), (8, 2, 128, 32), (3, 1, 256, 64), (2, 1, 32, 128), (4, 4, 96, 16)])
@pytest.mark.parametrize("fp8", [E4M3, E5M2])
def test_nan_in_keys_that_only_some_rows_see(seqs, H, Hk, D, P, fp8):
    """NaNs among the new tokens' keys and values reach the rows that see them, in the columns that hold them, and no others."""
    half = torch.bfloat16
    cu, T, lens = ranges(seqs)
    cache, table = filled(Hk, D, P, fp8, seqs, seed=30)
    for b, (n, s) in enumerate(seqs):
        for i, col in ((n - 1, 3), (n // 2, D - 1), (n // 2, 17), (max(0, n - 130), 0)):
            key = s - n + i
            cache[1][int(table[b, key // P]), 0, key % P, col] = math.nan
        key = s - n + n // 3
        cache[0][int(table[b, key // P]), Hk - 1, key % P, 7] = math.nan
    q = rows(T, H, D, half, 31, False, cu, seqs)
    where = to(DEV, table, lens, cu)
    out, lse = flash_attention_paged_kv(q, to(DEV, *cache), where[0], where[1], True, 0.1, cu_seqlens=where[2], return_lse=True)
    check_status(DEV)
    want, want_lse, A = po.attention(q.cpu(), cache, table, lens, True, 0.1, cu)
    got = out.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isnan(lse.cpu()), torch.isnan(want_lse))
    limit = torch.finfo(half).eps / 2 * want.abs() + 1.25 * 2.0 ** -11 * A + 2.0 ** -25
    held = ~torch.isnan(want)
    assert bool(((got - want).abs() <= limit)[held].all())


ITEMS = [(300, 300), (100, 500), (640, 640), (129, 700), (513, 1000), (90, 90), (257, 300), (20, 1200)]


@pytest.mark.parametrize("H,Hk,D,P", [(16, 16, 128, 64), (32, 16, 96, 16), (16, 16, 256, 32), (48, 24, 128, 128)])
@pytest.mark.parametrize("half,fp8", [(torch.float16, E4M3), (torch.bfloat16, E5M2)])
@pytest.mark.parametrize("far", [False, True], ids=["scales near", "scales far apart"])
def test_more_items_than_sms_of_which_some_have_one_tile(H, Hk, D, P, half, fp8, far):
    """CTAs that take over one item after another, where the last new tokens of a sequence fill no second tile of rows; with
    scales so far apart that they go through the softmax, which is slower, and without."""
    cu, T, lens = ranges(ITEMS)
    cache, table = filled(Hk, D, P, fp8, ITEMS, seed=80)
    if far:
        g = torch.Generator().manual_seed(81)
        for d, least in zip(cache[2:], (-30, -40)):
            d.copy_(torch.exp2(torch.randint(least, -7, d.shape, generator=g).float()))
    q = rows(T, H, D, half, 82, False, cu, ITEMS)
    where = to(DEV, table, lens, cu)
    out, lse = flash_attention_paged_kv(q, to(DEV, *cache), where[0], where[1], True, 0.05, cu_seqlens=where[2], return_lse=True)
    check_status(DEV)
    if not far:
        check_attention(q, cache, table, lens, True, 0.05, cu, out, lse)
        return
    # A probability (times its V's scale) below fp16's normal range is off by 2^-25 at most where the row's largest is 2^6 or more, so
    # n keys move a column by n 2^-25 448 / 2^6 of the largest value: less than 448 2^-25 of the row's largest sum, for n = 1200.
    want, want_lse, A = po.attention(q.cpu(), cache, table, lens, True, 0.05, cu)
    limit = torch.finfo(half).eps / 2 * want.abs() + 1.25 * 2.0 ** -11 * A + 448 * 2.0 ** -25 * A.amax(-1, keepdim=True) + 2.0 ** -25
    assert bool(((out.double().cpu() - want).abs() <= limit).all())
    assert bool(((lse.double().cpu() - want_lse).abs() <= 2.0 ** -20 * (want_lse.abs() + 16)).all())



@pytest.mark.parametrize("H,Hk,D,P", [(16, 16, 64, 64), (16, 8, 32, 16), (4, 4, 128, 32), (4, 2, 256, 16)])
@pytest.mark.parametrize("half,fp8", [(torch.float16, E4M3), (torch.bfloat16, E5M2)])
def test_scores_that_rise_from_block_to_block(H, Hk, D, P, half, fp8):
    """References are raised, and sums rescaled, at one block after another, in items of one tile and of two: a key's score is
    about 14 times one more than the number of its 128 keys."""
    seqs = [(100, 1000), (40, 700), (60, 60), (128, 129), (300, 900)] * (3 if D <= 64 else 1)
    cu, T, lens = ranges(seqs)
    cache, table = filled(Hk, D, P, fp8, seqs, seed=84)
    g = torch.Generator().manual_seed(86)
    for b, (_, s) in enumerate(seqs):
        for key in range(0, s, 16):                               # sixteen keys lie in one page
            row = torch.full((Hk, min(16, s - key), D), 1.0 + key // 128)
            row[:, :, 0] = torch.randint(0, 4, row.shape[:2], generator=g).float()
            cache[0][int(table[b, key // P]), :, key % P:key % P + row.shape[1]] = row.to(fp8)
        cache[2][table[b, :-(-s // P)].long()] = 1.0
    q = rows(T, H, D, half, 85, False, cu, seqs).abs()
    scale = 14 / (0.8 * D)                                        # the mean of a normal number's size is 0.8
    where = to(DEV, table, lens, cu)
    out, lse = flash_attention_paged_kv(q, to(DEV, *cache), where[0], where[1], True, scale, cu_seqlens=where[2], return_lse=True)
    check_status(DEV)
    check_attention(q, cache, table, lens, True, scale, cu, out, lse)


@pytest.mark.parametrize("seqs", [[(1, 20000), (1, 300)], [(3, 9000), (2, 12000)], [(1, 1500)], [(2, 700), (1, 40)], [(260, 3000)], [(150, 150), (300, 420)]],
                         ids=["tokens over CTAs", "drafts over CTAs", "a cluster", "clusters", "parts", "prompts"])
@pytest.mark.parametrize("H,Hk,D", [(4, 1, 128), (4, 2, 64), (2, 1, 256)])
def test_nan_in_queries(seqs, H, Hk, D):
    """A query row that holds a NaN is NaN, its log-sum-exp too, however its keys were shared out; the rows beside it are as they should be."""
    P, half = 64, torch.bfloat16
    cu, T, lens = ranges(seqs)
    cache, table = filled(Hk, D, P, E4M3, seqs, seed=90)
    q = rows(T, H, D, half, 91, False, cu, seqs)
    q[0, 1, 5] = math.nan
    q[T - 1, 0, D - 1] = math.nan
    q[T // 2, H - 1] = math.nan
    where = to(DEV, table, lens, cu)
    out, lse = flash_attention_paged_kv(q, to(DEV, *cache), where[0], where[1], True, 0.1, cu_seqlens=where[2], return_lse=True)
    check_status(DEV)
    want, want_lse, A = po.attention(q.cpu(), cache, table, lens, True, 0.1, cu)
    got, held = out.double().cpu(), ~torch.isnan(want)
    assert torch.equal(torch.isnan(got), ~held) and torch.equal(torch.isnan(lse.cpu()), torch.isnan(want_lse))
    limit = torch.finfo(half).eps / 2 * want.abs() + 1.25 * 2.0 ** -11 * A + 2.0 ** -25
    assert bool(((got - want).abs() <= limit)[held].all())


@pytest.mark.parametrize("S,Sk", [(256, 256), (4, 1024)], ids=["forward", "few rows"])
@pytest.mark.parametrize("op", ["append", "read", "attend"])
def test_an_index_out_of_range_leaves_the_calls_behind_it_alone(S, Sk, op):
    """A page out of range is left out of its own call and reported; a forward enqueued behind it, before anyone can know, is computed."""
    D = 64
    g = torch.Generator(device=DEV).manual_seed(100)
    q8, k8, v8 = (torch.randn(1, 2, s, D, generator=g, device=DEV).to(E4M3) for s in (S, Sk, Sk))
    want = flash_attention_v2_cutlass(q8, k8, v8, False, 0.125, v_layout="natural")[0]
    cache = PagedKVCache.empty(4, 2, D, 16, device=DEV)
    for t in cache:
        t.zero_()
    table, lens = torch.full((1, 2), 99, dtype=torch.int32, device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV)
    x, out = torch.zeros(3, 2, D, dtype=torch.float16, device=DEV), torch.full_like(want, 7.0)
    call = {"append": lambda t: paged_kv_append(cache, x, x, t, lens), "read": lambda t: paged_kv_read(cache, t, lens, 3),
            "attend": lambda t: flash_attention_paged_kv(x, cache, t, lens)}[op]
    call(torch.zeros_like(table))                                 # what a first call sets up is there
    check_status(DEV)
    torch.cuda._sleep(200_000_000)                                # a tenth of a second: the calls below are enqueued before the first has run
    call(table)
    flash_attention_v2_cutlass(q8, k8, v8, False, 0.125, v_layout="natural", out=out)
    with pytest.raises(RuntimeError, match="out of range"):
        check_status(DEV)
    assert torch.equal(bits(out), bits(want))
    check_status(DEV)


def test_an_expired_wait_behind_an_index_out_of_range_is_reported():
    lib, word = _lib.load(), api.status_word(DEV)
    cache = PagedKVCache.empty(4, 2, 64, 16, device=DEV)
    table, lens = torch.full((1, 2), 99, dtype=torch.int32, device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV)
    x = torch.zeros(3, 2, 64, dtype=torch.float16, device=DEV)
    paged_kv_append(cache, x, x, torch.zeros_like(table), lens)
    check_status(DEV)
    torch.cuda._sleep(200_000_000)
    paged_kv_append(cache, x, x, table, lens)
    assert lib.fa8_selftest_expired_wait(word.data_ptr(), 2000, torch.cuda.current_stream(DEV).cuda_stream) == _lib.FA8_OK
    with pytest.raises(RuntimeError, match="bounded wait"):
        check_status(DEV)
    check_status(DEV)


@pytest.mark.parametrize("seqs", [[(1, 300), (1, 90)], [(4, 300), (3, 3)], [(150, 500), (300, 300)]], ids=["tokens", "drafts", "prompts"])
@pytest.mark.parametrize("of", ["K", "V", "K and V"])
@pytest.mark.parametrize("H,Hk,D,fp8", [(4, 2, 64, E4M3), (4, 1, 128, E5M2), (2, 1, 256, E4M3), (4, 2, 96, E5M2)])
def test_first_pages_of_zeros_before_pages_of_the_largest_scale(seqs, of, H, Hk, D, fp8):
    """The scales that an append of zeros and of numbers past 2^70 leaves: 2^-64 on a sequence's first page, 2^64 on the others."""
    P, half = 16, torch.bfloat16
    cu, T, lens = ranges(seqs)
    cache, table = filled(Hk, D, P, fp8, seqs, seed=94)
    scale = 0.05
    for name, x8, d in (("K", cache[0], cache[2]), ("V", cache[1], cache[3])):
        if name in of:
            d.fill_(2.0 ** 64)
            for b, (_, s) in enumerate(seqs):
                x8[table[b, 0], :, :s] = 0.0
                d[table[b, 0]] = 2.0 ** -64
    if "K" in of:
        scale = 0.05 * 2.0 ** -70
    q = rows(T, H, D, half, 95, False, cu, seqs)
    where = to(DEV, table, lens, cu)
    out, lse = flash_attention_paged_kv(q, to(DEV, *cache), where[0], where[1], True, scale, cu_seqlens=where[2], return_lse=True)
    check_status(DEV)
    check_attention(q, cache, table, lens, True, scale, cu, out, lse)


@pytest.mark.parametrize("n,keys", [(1, 216), (4, 216), (150, 216), (1, 20000), (3, 9000), (150, 5000)])
@pytest.mark.parametrize("least", [2.0 ** -64, 0.0])
@pytest.mark.parametrize("H,Hk,D", [(1, 1, 64), (4, 1, 128), (16, 2, 256)])
def test_values_of_the_smallest_scale_still_count_in_the_denominators(n, keys, least, H, Hk, D):
    """Keys of a sequence with scores 6 below the other sixteen's, a third and more of the sum of exponentials, whose values are nothing beside
    the others': scales of V of 2^-64 (or nothing) and 2^64."""
    P, half = 16, torch.bfloat16
    seqs = [(n, keys + (n - 1) // 16 * 16)]
    cu, T, lens = ranges(seqs)
    cache, table = filled(Hk, D, P, E4M3, seqs, seed=96)
    cache[2].fill_(1.0)
    cache[3].fill_(least)
    cache[0].fill_(1.0)
    cache[3][table[0, 2]] = 2.0 ** 64
    cache[0][table[0, 2]] = 2.0
    cache[1].copy_(cache[1].float().nan_to_num(0.0).to(E4M3))
    q = rows(T, H, D, half, 97, False, cu, seqs).abs()
    q = q / q.float().sum(-1, keepdim=True).to(half)              # rows add up to about 1
    where = to(DEV, table, lens, cu)
    out, lse = flash_attention_paged_kv(q, to(DEV, *cache), where[0], where[1], False, 6.0, cu_seqlens=where[2], return_lse=True)
    check_status(DEV)
    check_attention(q, cache, table, lens, False, 6.0, cu, out, lse)


@pytest.mark.parametrize("n", [1, 5, 90])
@pytest.mark.parametrize("half,fp8", [(torch.float16, E4M3), (torch.bfloat16, E5M2), (torch.float16, E5M2)])
@pytest.mark.parametrize("D", [64, 256])
def test_append_to_pages_whose_scale_is_no_power_of_two(n, half, fp8, D):
    """Such a scale is kept where the new tokens fit it.  New values are odd numbers of half fp8 steps times 63 2^-7: they lie
    half-way between two fp8 numbers when divided by the scale, but not when multiplied by its rounded reciprocal."""
    Hk, P = 2, 128
    seqs = [(n, 20 + n), (n, 7 + n)]
    cu, T, lens = ranges(seqs)
    cache, table = filled(Hk, D, P, fp8, seqs, seed=98)
    for d in cache[2:]:
        d.fill_(63 * 2.0 ** -7)
    g = torch.Generator().manual_seed(99)
    mid = 2.0 * torch.randint(8, 16, (T, Hk, D), generator=g) + 1 if fp8 == E4M3 else 2.0 * torch.randint(4, 8, (T, Hk, D), generator=g) + 1
    x = (mid * 63 * 2.0 ** -7).to(half)
    exact = x.double() == mid.double() * 63 * 2.0 ** -7
    assert bool(exact.all()) or half is torch.bfloat16
    dev, where = PagedKVCache(*to(DEV, *cache)), to(DEV, table, lens)
    paged_kv_append(dev, x.to(DEV), -x.to(DEV), *where)
    check_status(DEV)
    for w, got in zip(po.append(cache, x, -x, table, lens), dev):
        assert torch.equal(w.float().nan_to_num(-1.0), got.cpu().float().nan_to_num(-1.0))


@pytest.mark.parametrize("seqs", [[(3, 40), (4, 300)], [(40, 200), (5, 5)], [(150, 500), (300, 300), (129, 140)], [(260, 3000)]], ids=["drafts", "pieces", "prompts", "parts"])
@pytest.mark.parametrize("H,Hk,D,P", [(2, 2, 64, 16), (8, 2, 128, 32), (3, 1, 256, 64), (2, 1, 32, 128)])
@pytest.mark.parametrize("half", [torch.float16, torch.bfloat16])
def test_infinities_in_keys_that_only_some_rows_see(seqs, H, Hk, D, P, half):
    """e5m2 has infinities.  Of V they reach the rows that see them, as an infinity or a NaN, in the columns that hold them, and
    leave the others alone; of K those whose scores they make infinite, as the definition has it."""
    cu, T, lens = ranges(seqs)
    cache, table = filled(Hk, D, P, E5M2, seqs, seed=92)
    for b, (n, s) in enumerate(seqs):
        for i, col, value in ((n - 1, 3, math.inf), (n // 2, D - 1, -math.inf), (n // 2, 17, math.inf), (n - 1, 17, -math.inf),
                              (max(0, n - 130), 0, math.inf), (n - 1, 0, math.nan)):
            key = s - n + i
            cache[1][int(table[b, key // P]), 0, key % P, col] = value
        if Hk > 1:                                                # in another head than V's
            key = s - n + n // 3
            cache[0][int(table[b, key // P]), Hk - 1, key % P, 7] = math.inf
    q = rows(T, H, D, half, 93, False, cu, seqs)
    where = to(DEV, table, lens, cu)
    out, lse = flash_attention_paged_kv(q, to(DEV, *cache), where[0], where[1], True, 0.1, cu_seqlens=where[2], return_lse=True)
    check_status(DEV)
    want, want_lse, A = po.attention(q.cpu(), cache, table, lens, True, 0.1, cu)
    got = out.double().cpu()
    held = torch.isfinite(want)
    assert bool(held.any()) and bool(torch.isinf(want).any())
    assert torch.equal(torch.isfinite(got), held)
    signed = torch.isinf(want) & torch.isinf(got)
    assert torch.equal(got[signed], want[signed])                 # never of the other sign
    assert bool(torch.isnan(got[torch.isnan(want)]).all())
    assert torch.equal(torch.isnan(lse.cpu()), torch.isnan(want_lse))
    limit = torch.finfo(half).eps / 2 * want.abs() + 1.25 * 2.0 ** -11 * A + 2.0 ** -25
    assert bool(((got - want).abs() <= limit)[held].all())


def test_page_table_of_wider_rows():
    """A view of a table that has more columns: as many as the longest sequence of this call needs."""
    seqs, H, Hk, D, P = [(1, 50), (1, 90), (1, 33)], 4, 2, 64, 16
    cu, T, lens = ranges(seqs)
    cache, table = filled(Hk, D, P, E4M3, seqs, seed=32)
    wide = torch.full((3, 40), -1, dtype=torch.int32)
    wide[:, 3:3 + table.shape[1]] = table
    q = rows(T, H, D, torch.float16, 33, False, cu, seqs)
    dev = to(DEV, *cache)
    a = flash_attention_paged_kv(q, dev, wide.to(DEV)[:, 3:9], lens.to(DEV), True, 0.1)[0]
    b = flash_attention_paged_kv(q, dev, table.to(DEV)[:, :6].contiguous(), lens.to(DEV), True, 0.1)[0]
    check_status(DEV)
    assert torch.equal(bits(a), bits(b))


@pytest.mark.parametrize("op", ["append", "read", "attend"])
@pytest.mark.parametrize("cu", [[0, 1000, 0, 8], [0, 2000, 1, 2], [5, 3, 2, 1], [0, 0, -9, 4]], ids=str)
@pytest.mark.parametrize("rows_of", [8, 1000])
def test_token_ranges_that_decrease_are_always_reported(op, cu, rows_of):
    """Also where no token is found to be of the sequence that has such a range."""
    T, Hk, D, P = rows_of, 2, 64, 16
    cache = PagedKVCache.empty(80, Hk, D, P, device=DEV)
    for t in cache:
        t.zero_()
    table = torch.arange(72, dtype=torch.int32, device=DEV).view(3, 24)
    lens = torch.full((3,), 300, dtype=torch.int32, device=DEV)
    where = dict(cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV))
    x = torch.ones(T, Hk, D, dtype=torch.float16, device=DEV)
    if op == "append":
        paged_kv_append(cache, x, x, table, lens, **where)
    elif op == "read":
        paged_kv_read(cache, table, lens, T, **where)
    else:
        flash_attention_paged_kv(x, cache, table, lens, True, 0.1, **where)
    with pytest.raises(RuntimeError, match="out of range"):
        check_status(DEV)
    check_status(DEV)


@pytest.mark.parametrize("n", [1, 4, 140])
def test_sequences_that_share_pages_and_rows_that_share_memory(n):
    """Two sequences with the same first pages; q, k and v whose rows or heads are one (strides of zero)."""
    H, Hk, D, P, half = 4, 2, 64, 16, torch.float16
    cache, table = filled(Hk, D, P, E4M3, [(n, 200 + n), (n, 200 + n)], seed=35)
    table[1, :12] = table[0, :12]                                 # 192 tokens
    lens = torch.tensor([200 + n] * 2, dtype=torch.int32)
    where = to(DEV, table, lens)
    g = torch.Generator().manual_seed(36)
    dev = PagedKVCache(*to(DEV, *cache))
    k = torch.randn(2 * n, 1, D, generator=g).to(half).to(DEV).expand(2 * n, Hk, D)
    v = torch.randn(1, Hk, D, generator=g).to(half).to(DEV).expand(2 * n, Hk, D)
    q = torch.randn(2 * n, 1, D, generator=g).to(half).to(DEV).expand(2 * n, H, D)
    paged_kv_append(dev, k, v, *where)
    after = po.append(cache, k.cpu(), v.cpu(), table, lens)
    for x, y in zip(dev, after):
        assert torch.equal(x.cpu().float().nan_to_num(-1.0), y.float().nan_to_num(-1.0))
    out, lse = flash_attention_paged_kv(q, dev, *where, True, 0.2, return_lse=True)
    check_status(DEV)
    check_attention(q, after, table, lens, True, 0.2, None, out, lse)


def test_offsets_past_32_bits_of_the_pool():
    """A pool of more than 2^32 bytes for K and for V, of which the last pages are used: as in a pool of those pages alone."""
    Hk, D, P, half, pages = 8, 128, 64, torch.bfloat16, 70000
    if torch.cuda.mem_get_info(DEV)[0] < 20 * 2 ** 30:
        pytest.skip("needs 20 GB")
    seqs = [(1, 300), (3, 70), (150, 150)]
    cu, T, lens = ranges(seqs)
    g = torch.Generator().manual_seed(37)
    big, small = PagedKVCache.empty(pages, Hk, D, P, device=DEV), PagedKVCache.empty(40, Hk, D, P, device=DEV)
    assert big.k.numel() > 2 ** 32
    table = torch.randperm(40, generator=g)[:15].view(3, 5).to(torch.int32)
    for t in small:
        t.zero_()
    for t in big:
        t[-40:].zero_()
    k, v, q = (torch.randn(T, h, D, generator=g).to(half).to(DEV) for h in (Hk, Hk, 4 * Hk))
    results = []
    for cache, first in ((small, 0), (big, pages - 40)):
        where = to(DEV, table + first, lens)
        paged_kv_append(cache, k, v, *where, cu_seqlens=cu.to(DEV))
        results.append([x[-40:] for x in cache] + list(paged_kv_read(cache, *where, T, cu_seqlens=cu.to(DEV), dtype=half))
                       + flash_attention_paged_kv(q, cache, *where, True, 0.1, cu_seqlens=cu.to(DEV)))
        results[-1] += flash_attention_paged_kv(q[:3], cache, *where, True, 0.1)
    check_status(DEV)
    for x, y in zip(*results):
        assert torch.equal(bits(x), bits(y))


def test_offsets_past_32_bits_of_the_rows():
    """More than 2^31 elements of rows: the last sequence's are those of a call of its own."""
    heads, D, P, half, n, B = 256, 128, 64, torch.float16, 10, 7000
    if torch.cuda.mem_get_info(DEV)[0] < 40 * 2 ** 30:
        pytest.skip("needs 40 GB")
    T = n * B
    x = torch.empty(T, heads, D, dtype=half, device=DEV)
    assert x.numel() > 2 ** 31
    x[:-4 * n].zero_()
    g = torch.Generator().manual_seed(38)
    x[-4 * n:] = torch.randn(4 * n, heads, D, generator=g).to(half).to(DEV)
    cache = PagedKVCache.empty(B, heads, D, P, device=DEV)
    table = torch.arange(B, dtype=torch.int32, device=DEV).view(B, 1)
    lens = torch.full((B,), n, dtype=torch.int32, device=DEV)
    paged_kv_append(cache, x, x, table, lens)
    alone = PagedKVCache.empty(4, heads, D, P, device=DEV)
    paged_kv_append(alone, x[-4 * n:], x[-4 * n:], table[:4], lens[:4])
    for a, b in zip(cache, alone):
        a, b = (a[-4:], b) if a.dim() == 2 else (a[-4:, :, :n], b[:, :, :n])
        assert torch.equal(bits(a), bits(b))
    got = paged_kv_read(cache, table, lens, T, dtype=half)
    want = paged_kv_read(alone, table[:4], lens[:4], 4 * n, dtype=half)
    assert torch.equal(bits(got[0][-4 * n:]), bits(want[0])) and torch.equal(bits(got[1][-4 * n:]), bits(want[1]))
    del got
    out = flash_attention_paged_kv(x, cache, table, lens, True, 0.1)[0]
    check_status(DEV)
    last = x[-n:].cpu()
    o, _, A = po.attention(last, [t.cpu() for t in alone], table[3:4].cpu(), lens[:1].cpu(), True, 0.1)
    assert bool(((out[-n:].double().cpu() - o).abs() <= torch.finfo(half).eps / 2 * o.abs() + 1.25 * 2.0 ** -11 * A + 2.0 ** -25).all())
    assert not bool(out[:-4 * n].any())


# ---- a run of them, graphs, streams ---------------------------------------------------------------------------

def test_generation_step_by_step_and_read_back():
    """Prompts are appended and attended to, then tokens one at a time; whole sequences are read back at the end."""
    H, Hk, D, P, half = 8, 2, 128, 16, torch.bfloat16
    prompts, steps = [37, 5, 64], 30
    B = len(prompts)
    total = [p + steps for p in prompts]
    need = [-(-t // P) for t in total]
    cache = PagedKVCache.empty(sum(need), Hk, D, P, device=DEV)
    table = torch.full((B, max(need)), -1, dtype=torch.int32)
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    table_d = table.to(DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    scale = 1 / math.sqrt(D)
    host = [t.cpu() for t in cache]
    lens = torch.tensor(prompts, dtype=torch.int32)
    cu = torch.tensor([0] + prompts).cumsum(0).to(torch.int32)
    for step in range(steps + 1):
        T = int(cu[-1]) if step == 0 else B
        qkv = torch.randn(T, H + 2 * Hk, D, generator=g, device=DEV).to(half)
        q, k, v = qkv.split((H, Hk, Hk), 1)
        c = cu if step == 0 else None
        lens_d, c_d = lens.to(DEV), None if c is None else c.to(DEV)
        paged_kv_append(cache, k, v, table_d, lens_d, cu_seqlens=c_d)
        out, lse = flash_attention_paged_kv(q, cache, table_d, lens_d, True, scale, cu_seqlens=c_d, return_lse=True)
        host = po.append(host, k.cpu(), v.cpu(), table, lens, c)
        if step in (0, 1, 12, steps):
            check_attention(q, host, table, lens, True, scale, c, out, lse)
        if step < steps:
            lens = lens + 1
    check_status(DEV)
    every = lens.cumsum(0)
    cu_all = torch.cat([torch.zeros(1, dtype=torch.int32), every.to(torch.int32)])
    T = int(every[-1])
    for w, got in zip(po.read(host, table, lens, T, cu_all), paged_kv_read(cache, table_d, lens.to(DEV), T, cu_seqlens=cu_all.to(DEV), dtype=half)):
        assert torch.equal(bits(w.to(half)), bits(got))
    check_status(DEV)


def captured(f):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        f()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = f()
    return graph, r


@pytest.mark.parametrize("n", [1, 3, 140])
def test_captured_steps_replay_with_other_lengths(n):
    H, Hk, D, P, B, half = 8, 2, 64, 16, 3, torch.float16
    width = 60
    cache = PagedKVCache.empty(B * width, Hk, D, P, device=DEV)
    for t in cache:
        t.zero_()
    table = torch.arange(B * width, dtype=torch.int32).view(B, width)
    lens_d = torch.full((B,), n, dtype=torch.int32, device=DEV)
    table_d = table.to(DEV)
    q, k, v = (torch.zeros(B * n, h, D, dtype=half, device=DEV) for h in (H, Hk, Hk))

    def step():
        paged_kv_append(cache, k, v, table_d, lens_d)
        return flash_attention_paged_kv(q, cache, table_d, lens_d, True, 0.2, return_lse=True)

    graph, (out, lse) = captured(step)
    host = [t.cpu() for t in cache]
    g = torch.Generator(device=DEV).manual_seed(8)
    lens = torch.zeros(B, dtype=torch.int32)
    for grow in ([n, n, n], [n, n + 40, n], [n + 300, n, n + 1]):
        lens = lens + torch.tensor(grow, dtype=torch.int32)      # tokens skipped over: pages keep what they held
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        lens_d.copy_(lens)
        host = po.append(host, k.cpu(), v.cpu(), table, lens)
        graph.replay()
        check_status(DEV)
        for w, c in zip(host, cache):
            assert torch.equal(w.float(), c.cpu().float())
        check_attention(q, host, table, lens, True, 0.2, None, out, lse)


def test_two_captured_calls_at_once():
    """Two graphs of long attention calls on two streams at the same time: each has a workspace of its own."""
    seqs = [(1, 5000)]
    H, Hk, D, P = 8, 2, 128, 64
    graphs, outs, alone = [], [], []
    keep = []
    for i in range(2):
        cache, table = filled(Hk, D, P, E4M3, seqs, seed=20 + i)
        q = rows(1, H, D, torch.float16, 30 + i, False, None, seqs)
        args = (q, to(DEV, *cache), table.to(DEV), torch.tensor([5000], dtype=torch.int32, device=DEV), True, 0.1)
        keep.append(args)
        alone.append(flash_attention_paged_kv(*args)[0].clone())
        graph, r = captured(lambda: flash_attention_paged_kv(*args))
        graphs.append(graph)
        outs.append(r[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(50):
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    check_status(DEV)
    for o, a in zip(outs, alone):
        assert torch.equal(o, a)


def test_another_stream_than_the_current_one_of_the_tensors():
    seqs = [(3, 200)]
    want = attend(seqs, 4, 2, 64, 16, torch.float16, E4M3, True, seed=40)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = attend(seqs, 4, 2, 64, 16, torch.float16, E4M3, True, seed=40)
    assert torch.equal(want, got)


def test_the_same_call_twice_gives_the_same_bits():
    for seqs in ([(1, 4000), (1, 77)], [(300, 2000)]):
        a, b = (attend(seqs, 8, 2, 128, 16, torch.bfloat16, E4M3, True, seed=50) for _ in range(2))
        assert torch.equal(a, b)


# ---- numbers out of range -------------------------------------------------------------------------------------

@pytest.mark.parametrize("what", ["page too large", "page negative", "length negative", "length too large", "more new than held", "range decreases", "range ends outside"])
@pytest.mark.parametrize("op", ["append", "read", "attend one", "attend many"])
def test_numbers_out_of_range_are_left_out_and_reported(what, op):
    n = 150 if op == "attend many" else 1
    if what.startswith("more") and op.startswith("attend"):
        pytest.skip("such rows see no key")
    H, Hk, D, P = 4, 2, 64, 16
    seqs = [(n, n + 40), (n, n + 70), (n, n + 3)]
    cache, table = filled(Hk, D, P, E4M3, seqs, seed=60)
    table[0, -2:] = 0
    cu = torch.tensor([0, n, 2 * n, 3 * n], dtype=torch.int32)
    lens = torch.tensor([s for _, s in seqs], dtype=torch.int32)
    good = po.attention(rows(3 * n, H, D, torch.float16, 61, False, cu, seqs).cpu(), cache, table, lens, True, 0.1, cu)
    at = -(-(n + 70) // P) - 1
    if what == "page too large":
        table[1, at] = cache[0].shape[0]
    elif what == "page negative":
        table[1, at] = -1
    elif what == "length negative":
        lens[1] = -5
    elif what == "length too large":
        lens[1] = table.shape[1] * P + 1
    elif what == "more new than held":
        lens[1] = n - 1
    elif what == "range decreases":
        cu[3] = 2 * n - 1
    else:
        cu[3] = 3 * n + 1
    dev, table_d, lens_d, cu_d = PagedKVCache(*to(DEV, *cache)), *to(DEV, table, lens, cu)
    q, k, v = (rows(3 * n, h, D, torch.float16, s, False, None, seqs) for h, s in ((H, 61), (Hk, 62), (Hk, 63)))

    def call():
        if op == "append":
            paged_kv_append(dev, k, v, table_d, lens_d, cu_seqlens=cu_d)
            return None
        if op == "read":
            return paged_kv_read(dev, table_d, lens_d, 3 * n, cu_seqlens=cu_d)
        return flash_attention_paged_kv(q, dev, table_d, lens_d, True, 0.1, cu_seqlens=cu_d)

    got = call()
    with pytest.raises(RuntimeError, match="out of range"):
        check_status(DEV)
    check_status(DEV)                                             # reported once
    call()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="out of range"):       # without check_status the next call says so
        call()
    torch.cuda.synchronize()
    api.status_word(DEV).zero_()
    check_status(DEV)
    # the first sequence is as it should be
    if op.startswith("attend"):
        limit = torch.finfo(torch.float16).eps / 2 * good[0][:n].abs() + 1.25 * 2.0 ** -11 * good[2][:n] + 2.0 ** -25
        assert bool(((got[0][:n].double().cpu() - good[0][:n]).abs() <= limit).all())
        if what.startswith("length"):
            assert bool((got[0][n:2 * n] == 0).all())
        assert what.startswith("range") or bool(torch.isfinite(got[0]).all())
    elif op == "read":
        want = po.read(cache, table, lens[:1], n, cu[:2])
        assert torch.equal(got[0][:n].double().cpu(), want[0])
        if what.startswith(("page", "length", "more")):
            assert bool((got[0][n:2 * n] == 0).all())
    else:
        want = po.append(cache, k[:n].cpu(), v[:n].cpu(), table, lens[:1], cu[:2])
        page = int(table[0, (n + 39) // P])
        assert torch.equal(want[0][page].float().nan_to_num(-1.0), dev.k.cpu()[page].float().nan_to_num(-1.0))


# ---- refusals ---------------------------------------------------------------------------------------------------

def good_call():
    cache = PagedKVCache.empty(6, 2, 64, 16, device=DEV)
    for t in cache:
        t.zero_()
    return dict(cache=cache, q=torch.zeros(2, 4, 64, dtype=torch.float16, device=DEV), k=torch.zeros(2, 2, 64, dtype=torch.float16, device=DEV),
                v=torch.zeros(2, 2, 64, dtype=torch.float16, device=DEV), table=torch.arange(6, dtype=torch.int32, device=DEV).view(2, 3),
                seqlens=torch.tensor([1, 20], dtype=torch.int32, device=DEV), cu=None, scale=0.1, out=None)


def refused(match, ops=("append", "read", "attend"), **kw):
    a = {**good_call(), **kw}
    for op in ops:
        with pytest.raises(RuntimeError, match=match):
            if op == "append":
                paged_kv_append(a["cache"], a["k"], a["v"], a["table"], a["seqlens"], cu_seqlens=a["cu"])
            elif op == "read":
                paged_kv_read(a["cache"], a["table"], a["seqlens"], a.get("tokens", 2), cu_seqlens=a["cu"], dtype=a.get("dtype", torch.float16))
            else:
                flash_attention_paged_kv(a["q"], a["cache"], a["table"], a["seqlens"], True, a["scale"], cu_seqlens=a["cu"], out=a["out"])


def test_refusals():
    c = good_call()["cache"]
    cpu = [t.cpu() for t in c]
    refused("CUDA", cache=[cpu[0], *c[1:]])
    refused("CUDA", cache=[*c[:3], cpu[3]])
    refused("contiguous", cache=[c.k.transpose(0, 1), *c[1:]])
    refused("float8", cache=[c.k.view(torch.uint8), *c[1:]])
    refused("float8", cache=[c.k, c.v.view(E5M2), *c[2:]])
    refused("alike", cache=[c.k, c.v[:5], *c[2:]])
    refused("no pages", cache=[c.k[:0], c.v[:0], c.k_descale[:0], c.v_descale[:0]])
    refused("page_size", cache=[c.k.view(6, 2, 8, 128), c.v.view(6, 2, 8, 128), *c[2:]])
    refused("head_dim", cache=[c.k.view(6, 2, 64, 16), c.v.view(6, 2, 64, 16), *c[2:]])
    refused("k_descale", cache=[*c[:2], c.k_descale.double(), c.v_descale])
    refused("v_descale", cache=[*c[:3], c.v_descale[:, :1].contiguous()])
    t, s = good_call()["table"], good_call()["seqlens"]
    refused("page_table", table=t.long())
    refused("page_table", table=t.cpu())
    refused("page_table", table=t[:1])
    refused("page_table", table=t.t().contiguous().t())
    refused("page_table", table=torch.zeros(1, 3, dtype=torch.int32, device=DEV).expand(2, 3))
    refused("seqlens", seqlens=s.long())
    refused("seqlens", seqlens=s.view(1, 2))
    refused("seqlens", seqlens=torch.zeros(4, dtype=torch.int32, device=DEV)[::2])
    refused("cu_seqlens", cu=s)
    refused("cu_seqlens", cu=torch.zeros(3, dtype=torch.int64, device=DEV))
    refused("no pages to hold", table=t[:, :0])
    refused("evenly", ops=("read",), tokens=3)
    refused("number of rows", ops=("read",), tokens=-2)
    refused("dtype", ops=("read",), dtype=torch.float32)
    k = good_call()["k"]
    refused("float16", ops=("append",), k=k.float(), v=k.float())
    refused("same type", ops=("append",), v=k.bfloat16())
    refused("same type", ops=("append",), v=k[:1])
    refused("k must be", ops=("append",), k=k[:, :1])
    refused("k must be", ops=("append",), k=torch.zeros(2, 2, 96, dtype=torch.float16, device=DEV))
    refused("16 bytes", ops=("append",), k=torch.zeros(2 * 2 * 64 + 4, dtype=torch.float16, device=DEV)[4:].view(2, 2, 64))
    refused("16 bytes", ops=("append",), k=torch.zeros(2, 64, 2, dtype=torch.float16, device=DEV).transpose(1, 2))
    refused("gradient", ops=("append",), k=k.clone().requires_grad_())
    q = good_call()["q"]
    refused("gradient", ops=("attend",), q=q.clone().requires_grad_())
    refused("multiple", ops=("attend",), q=q[:, :3])
    refused("q must be", ops=("attend",), q=q[0])
    refused("float16", ops=("attend",), q=q.float())
    refused("out must", ops=("attend",), out=torch.empty(2, 4, 64, dtype=torch.bfloat16, device=DEV))
    refused("contiguous", ops=("attend",), out=torch.empty(2, 64, 4, dtype=torch.float16, device=DEV).transpose(1, 2))
    for bad in (0.0, -1.0, math.nan, math.inf):
        refused("bad argument", ops=("attend",), scale=bad)
    check_status(DEV)
    with torch.no_grad():
        a = good_call()
        flash_attention_paged_kv(q.clone().requires_grad_(), a["cache"], a["table"], a["seqlens"], True, 0.1)
    check_status(DEV)


def test_no_tokens():
    a = good_call()
    empty = a["k"][:0]
    paged_kv_append(a["cache"], empty, empty, a["table"], a["seqlens"])
    k, v = paged_kv_read(a["cache"], a["table"], a["seqlens"], 0)
    assert k.shape == v.shape == (0, 2, 64)
    assert flash_attention_paged_kv(a["q"][:0], a["cache"], a["table"], a["seqlens"])[0].shape == (0, 4, 64)
    check_status(DEV)


def test_through_the_module_and_through_ctypes(monkeypatch):
    native = api._native()
    assert native
    seqs = [(2, 33), (5, 90)]
    cu, T, lens = ranges(seqs)
    cache, table = filled(2, 64, 16, E4M3, seqs, seed=70)
    q, k, v = (rows(T, h, 64, torch.bfloat16, s, True, None, seqs) for h, s in ((6, 71), (2, 72), (2, 73)))
    results = []
    for module in (native, False):
        taken = []

        class Counting:
            def __getattr__(self, name):
                def through(*a):
                    r = getattr(module, name)(*a)
                    taken.append(r)
                    return r
                return through

        monkeypatch.setattr(api, "_native_module", Counting() if module else False)
        dev, tables = PagedKVCache(*to(DEV, *cache)), to(DEV, table, lens, cu)
        paged_kv_append(dev, k, v, tables[0], tables[1], cu_seqlens=tables[2])
        got = list(paged_kv_read(dev, tables[0], tables[1], T, cu_seqlens=tables[2], dtype=torch.bfloat16))
        got += flash_attention_paged_kv(q, dev, tables[0], tables[1], True, 0.3, cu_seqlens=tables[2], return_lse=True)
        check_status(DEV)
        assert len(taken) == (3 if module else 0) and all(r is not None for r in taken)
        results.append([bits(t) for t in (*dev, *got)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
