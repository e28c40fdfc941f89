"""The 8-bit paged KV cache on the GPU against plain forms in 64 bits."""
import math

import pytest
import torch

import picolm_b200 as pb
from tests.kv8_util import (BLOCK, DTYPES, PAGE, TOP, TORCH, Cache, attention_bound, generator, i32, randn, rotate,
                            starts, stream)

pytestmark = pytest.mark.gpu
FORMATS = (pb.PL_KV8_INT8, pb.PL_KV8_E4M3)


# ------------------------------------------------------------------ append
def check_rows(c, slot, first, rows, x, kv, layer=0):
    """Rows [first, first + len(x)) of a slot hold x to half a step.

    int8: |code - x / s| <= 1/2, with x / s off by the division's rounding
    and, for k, the rotation's (8u of the block's largest value, 127 s):
    (1/2 + 127 * 9 * 2^-24) s.  e4m3: half a step is 2^-4 of the value,
    or 2^-10 below the smallest normal 2^-6: max(|x| 2^-4, 2^-10 s) and the same slack."""
    got = c.values(slot, rows, layer)[kv][first:first + len(x)]
    pages = c.table[slot, :-(-rows // PAGE)].long()
    s = c.scales[pages, layer][:, :, kv].double()                       # [page][head][block]
    s = s.permute(0, 2, 1).reshape(-1, c.kv_heads).repeat_interleave(BLOCK, 0)[first:first + len(x), :, None]
    slack = TOP[c.fmt] * 9 * 2.0 ** -24 * s
    half = 0.5 * s if c.fmt == pb.PL_KV8_INT8 else torch.maximum(x.abs() / 16, s * 2.0 ** -10)
    assert bool(((got - x).abs() <= half + slack).all())
    return s


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("head_dim,layout,dim", [(64, pb.PL_ROPE_LLAMA, 64), (128, pb.PL_ROPE_QWEN, 128),
                                                 (64, pb.PL_ROPE_QWEN, 36), (128, pb.PL_ROPE_LLAMA, 10),
                                                 (64, pb.PL_ROPE_LLAMA, 0)])
def test_append_whole_blocks_and_tails(fmt, dtype, head_dim, layout, dim):
    gen = generator(1)
    counts = [1, 15, 16, 17, 64, 65, 130]
    c = Cache(6, 3, head_dim, fmt, n_pages=16, n_seqs=8, max_pages=4, layers=2, layout=layout, rope_dim=dim)
    seqs = [6, 0, 3, 1, 7, 2, 4]
    c.resize(seqs, counts)
    before = c.codes.clone()
    rows = randn(gen, sum(counts), 2 * 3 * head_dim + 16, dtype=TORCH[dtype])
    k, v = rows[:, :3 * head_dim], rows[:, 3 * head_dim:6 * head_dim]
    c.append(seqs, counts, k, v, dtype, layer=1)
    st = starts(counts)
    for i, (slot, n) in enumerate(zip(seqs, counts)):
        kr = rotate(k[st[i]:st[i + 1]].reshape(n, 3, head_dim), torch.arange(n, device="cuda"), c.freq, c.gain, layout)
        vr = v[st[i]:st[i + 1]].double().reshape(n, 3, head_dim)
        for kv, x in ((0, kr), (1, vr)):
            s = check_rows(c, slot, 0, n, x, kv, layer=1)
            for b in range(0, n, BLOCK):  # the scale is the block's largest value over the largest code
                want = x[b:b + BLOCK].abs().amax((0, 2)) / TOP[fmt]
                assert torch.allclose(s[b, :, 0], want, rtol=10 * 2.0 ** -24, atol=0)
    # the other layer, free pages and rows past the end keep what they held
    assert torch.equal(c.codes[:, 0], before[:, 0])
    for slot, n in zip(seqs, counts):
        if n % PAGE:
            p = int(c.table[slot, n // PAGE])
            assert torch.equal(c.codes[p, 1, :, :, n % PAGE:], before[p, 1, :, :, n % PAGE:])
    free = c.refs == 0
    assert torch.equal(c.codes[free], before[free])


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_rescales_the_rows_of_its_block(fmt):
    gen = generator(2)
    c = Cache(4, 2, 64, fmt)
    c.resize([0], [5])
    k, v = randn(gen, 5, 128), randn(gen, 5, 128)
    c.append([0], [5], k, v, pb.PL_F32)
    old, old_s = c.values(0, 5).clone(), c.scales[int(c.table[0, 0]), 0, :, :, 0].clone()
    codes = c.codes[int(c.table[0, 0]), 0, :, :, :5].clone()
    c.resize([0], [6])
    small = torch.zeros(1, 128, device="cuda")
    c.append([0], [1], small, small, pb.PL_F32)  # a smaller row leaves the block as it is
    assert torch.equal(c.codes[int(c.table[0, 0]), 0, :, :, :5], codes)
    assert torch.equal(c.scales[int(c.table[0, 0]), 0, :, :, 0], old_s)
    c.resize([0], [7])
    big = torch.full((1, 128), 50.0, device="cuda")
    c.append([0], [1], big, big, pb.PL_F32)
    s = c.scales[int(c.table[0, 0]), 0, :, :, 0].double()
    assert bool((s > old_s).all())
    err = (c.values(0, 5) - old).abs()
    half = (0.5 * s.t()[:, None, :, None] if fmt == pb.PL_KV8_INT8
            else torch.maximum(old.abs() / 16, s.t()[:, None, :, None] * 2.0 ** -10))
    assert bool((err <= half * (1 + 2.0 ** -15)).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_of_zeros_and_of_nonfinite_rows(fmt):
    c = Cache(2, 2, 64, fmt)
    c.resize([0, 1], [3, 20])
    z = torch.zeros(23, 128, device="cuda")
    z[3 + 18, 0] = math.inf   # slot 1, second block, head 0
    z[3 + 2, 64] = math.nan   # slot 1, first block, head 1
    c.append([0, 1], [3, 20], z, torch.zeros_like(z), pb.PL_F32)
    assert bool((c.values(0, 3) == 0).all())
    k, v = c.values(1, 20)
    assert bool((v == 0).all())
    assert bool(torch.isnan(k[16:, 0]).all()) and bool((k[:16, 0] == 0).all())
    assert bool(torch.isnan(k[:16, 1]).all()) and bool((k[16:, 1] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_read_back(fmt, dtype):
    gen = generator(3)
    c = Cache(4, 4, 128, fmt, n_seqs=3)
    c.fill([2, 0], [130, 70], gen)
    row0, counts = [3, 69, 0], [127, 1, 0]
    k = torch.full((130, 4 * 128 + 8), 7.0, dtype=TORCH[dtype], device="cuda")
    v = k.clone()
    a, b, st = i32([2, 0, 1]), i32(row0), i32(starts(counts))
    c.c.read_dev(0, 3, a.data_ptr(), b.data_ptr(), st.data_ptr(), 128, 127, dtype, k.data_ptr(), k.stride(0),
                 v.data_ptr(), v.stride(0), stream())
    assert c.c.status(stream()) == pb.PL_OK
    want = torch.cat((c.values(2, 130)[:, 3:130], c.values(0, 70)[:, 69:70]), 1).reshape(2, 128, -1)
    # code * scale in FP32 (u = 2^-24), then one rounding to the type
    tol = 2.0 ** -24 + (0 if dtype == pb.PL_F32 else torch.finfo(TORCH[dtype]).eps / 2 * (1 + 2.0 ** -10))
    tiny = torch.finfo(TORCH[dtype]).tiny
    for got, x in ((k, want[0]), (v, want[1])):
        assert bool(((got[:128, :512].double() - x).abs() <= tol * x.abs() + tiny).all())
        assert bool((got[128:] == 7).all()) and bool((got[:, 512:] == 7).all())


# --------------------------------------------------------------- attention
def attend_and_check(c, seqs, counts, dtype, gen, layer=0, q_scale=1.0):
    total = sum(counts)
    wide = randn(gen, total + 3, c.heads * c.head_dim + 16, dtype=TORCH[dtype])
    q = (wide[:, :c.heads * c.head_dim] * q_scale).to(TORCH[dtype])
    rows = torch.full((total + 3, c.heads * c.head_dim + 24), 7.0, dtype=TORCH[dtype], device="cuda")
    out = rows[:, 8:8 + c.heads * c.head_dim]
    c.attend(seqs, counts, q, out, dtype, layer)
    want, most, vmax = c.reference(seqs, counts, q, layer)
    err = (out[:total].double() - want).abs()
    bound = attention_bound(dtype, c.head_dim, int(c.lens.max()), most, vmax, want)
    assert bool((err <= bound).all()), float((err - bound).max())
    assert bool((rows[total:] == 7).all()) and bool((rows[:, :8] == 7).all()) and bool((rows[:, -16:] == 7).all())
    return out[:total], want


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("group,kv_heads", [(1, 3), (7, 2), (8, 1), (4, 4)])
def test_one_token_at_every_kind_of_length(fmt, head_dim, group, kv_heads):
    gen = generator(4)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 100, 127, 128, 129, 192, 447, 511, 512]
    c = Cache(group * kv_heads, kv_heads, head_dim, fmt, n_pages=64, n_seqs=len(lens), max_pages=8)
    order = [int(i) for i in torch.randperm(len(lens), generator=torch.Generator().manual_seed(1))]
    c.fill(order, lens, gen)
    for dtype in DTYPES:
        attend_and_check(c, order, [1] * len(lens), dtype, gen)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("head_dim,layout", [(64, pb.PL_ROPE_LLAMA), (128, pb.PL_ROPE_QWEN)])
@pytest.mark.parametrize("counts,lens", [
    ([2, 3, 5], [2, 70, 300]), ([17, 1, 0, 64], [17, 200, 33, 64]), ([128, 127, 129], [128, 400, 129]),
    ([300], [512]), ([200, 256], [201, 256]), ([31, 33, 16, 47], [500, 65, 16, 512])])
def test_several_tokens(fmt, head_dim, layout, counts, lens):
    gen = generator(5)
    c = Cache(8, 2, head_dim, fmt, n_pages=64, n_seqs=len(lens) + 1, max_pages=8, layout=layout)
    seqs = list(range(len(lens), 0, -1))
    c.fill(seqs, lens, gen)
    for dtype in DTYPES:
        attend_and_check(c, seqs, counts, dtype, gen)


@pytest.mark.parametrize("group,kv_heads", [(1, 1), (3, 2), (5, 1), (6, 1), (7, 4), (8, 2), (2, 8)])
def test_several_tokens_of_every_group(group, kv_heads):
    gen = generator(6)
    c = Cache(group * kv_heads, kv_heads, 64, n_pages=32, n_seqs=2, max_pages=8)
    c.fill([0, 1], [333, 150], gen)
    for dtype in (pb.PL_F32, pb.PL_BF16):
        attend_and_check(c, [1, 0], [150, 77], dtype, gen)


@pytest.mark.parametrize("counts,lens", [([1, 1], [0, 5]), ([4, 6, 3], [2, 0, 3]), ([150, 200], [20, 130])])
def test_tokens_with_no_row_to_attend_are_zero(counts, lens):
    """More query tokens than rows: the first ones see nothing."""
    gen = generator(7)
    c = Cache(8, 2, 64, n_seqs=len(lens))
    c.fill(list(range(len(lens))), lens, gen)
    for dtype in DTYPES:
        out, _ = attend_and_check(c, list(range(len(lens))), counts, dtype, gen)
        t = 0
        for n, m in zip(counts, lens):
            assert bool((out[t:t + max(0, n - m)] == 0).all())
            t += n


@pytest.mark.parametrize("count", [1, 40])
def test_large_and_small_magnitudes(count):
    """Scores far from 0 (one row takes all) and values far from 1: q of 1e5
    and of 1e-6, k and v blocks from 1e-8 to 1e8."""
    gen = generator(8)
    c = Cache(8, 2, 64, n_seqs=1, n_pages=16)
    c.fill([0], [300], gen)
    pages = c.table[0, :5].long()
    c.scales[pages, 0, :, 1] *= torch.logspace(-8, 8, 20, device="cuda").view(5, 1, 4)
    for q_scale in (1.0, 1e-6, 1e5):
        attend_and_check(c, [0], [count], pb.PL_F32, gen, q_scale=q_scale)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("length", [100, 320])
def test_later_values_do_not_reach_earlier_tokens(fmt, head_dim, length):
    """A prompt whose V scales rise from block to block: the masked blocks of
    a tile are up to 10^13 times larger than the ones that a token sees.

    attention_bound holds with each token's own largest |v|, the largest
    scale of the blocks that it sees times the largest code: a weight in two
    FP16 parts is off by 2^-25 at least, in units of which the largest visible
    scale is 16 to 64, so by no more than `rows` 2^-29 of that |v| over all
    rows, which the bound's 2 rows 2^-24 covers."""
    gen = generator(31)
    c = Cache(8, 2, head_dim, fmt, n_pages=32, n_seqs=1, max_pages=16)
    c.fill([0], [length], gen)
    pages = c.table[0, :-(-length // PAGE)].long()
    for dtype, lo, hi in ((pb.PL_F32, -20, 12), (pb.PL_BF16, -20, 12), (pb.PL_F16, -5, 2)):
        saved = c.scales.clone()
        rise = torch.linspace(lo, hi, 4 * len(pages), device="cuda").view(-1, 1, 4)
        c.scales[pages, 0, :, 1] *= 10.0 ** rise
        q = randn(gen, length, 8 * head_dim, dtype=TORCH[dtype])
        out = c.attend([0], [length], q, torch.empty_like(q), dtype)
        want, most, _ = c.reference([0], [length], q)
        top = c.scales[pages, 0, :, 1].permute(1, 0, 2).reshape(2, -1).double()  # [kv head][block]
        top = torch.nan_to_num(top, 0.0).cummax(1).values * TOP[fmt]
        vmax = top.repeat_interleave(BLOCK, 1)[:, :length].t()                   # [token][kv head]
        vmax = vmax.repeat_interleave(4 * head_dim, 1)
        err = (out.double() - want).abs()
        assert bool((err <= attention_bound(dtype, head_dim, length, most, vmax, want)).all()), float(
            (err / vmax).max())
        c.scales.copy_(saved)


def test_nan_stays_where_it_is():
    """A NaN block is seen by tokens that attend it, by no others; a NaN in q
    by its own head and token."""
    gen = generator(9)
    c = Cache(4, 2, 64, n_seqs=2)
    c.fill([0, 1], [100, 100], gen)
    c.scales[int(c.table[0, 1]), 0, 1, 0, 1] = math.nan   # rows 80..95, head 1, K
    q = randn(gen, 200, 256)
    q[150, 0] = math.nan
    out = c.attend([0, 1], [100, 100], q, torch.empty_like(q), pb.PL_F32).view(200, 4, 64)
    bad = torch.isnan(out).any(-1)
    want = torch.zeros(200, 4, dtype=torch.bool, device="cuda")
    want[80:100, 2:] = True
    want[150, 0] = True
    assert torch.equal(bad, want)
    # the same for V, and one token at a time
    c.scales[int(c.table[0, 1]), 0, 1, 0, 1] = 0.02
    c.scales[int(c.table[0, 1]), 0, 0, 1, 1] = math.nan   # rows 80..95, head 0, V
    q[150, 0] = 1.0
    out = c.attend([0, 1], [100, 100], q, torch.empty_like(q), pb.PL_F32).view(200, 4, 64)
    want[:] = False
    want[80:100, :2] = True
    assert torch.equal(torch.isnan(out).any(-1), want)
    out = c.attend([0, 1], [1, 1], q[:2], torch.empty_like(q[:2]), pb.PL_F32).view(2, 4, 64)
    assert torch.isnan(out).any(-1).tolist() == [[True, True, False, False], [False] * 4]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("one", [False, True], ids=["append", "decode"])
def test_appended_nonfinite_values_reach_no_earlier_token(fmt, head_dim, value, one):
    """Rows 80..95 share a scale; row 85 of V (head 0) or of K (head 1) is
    not finite, appended with the others or by a decode step.  Tokens from
    row 80 on are NaN in that head; the others are as over a cache that had
    0 there."""
    gen = generator(32)
    kd, n = 2 * head_dim, 86 if one else 100
    k, v, q = (randn(gen, n, w) for w in (kd, kd, 2 * kd))
    k[85, head_dim + 3] = v[85, 5] = 0
    caches = []
    for bad in (value, 0.0):
        c = Cache(4, 2, head_dim, fmt, n_seqs=1)
        k[85, head_dim + 3] = v[85, 5] = bad
        first = 85 if one else 100
        c.resize([0], [first])
        c.append([0], [first], k[:first], v[:first], pb.PL_F32)
        if one:
            c.resize([0], [86])
            out = c.decode([0], q[85:], k[85:], v[85:], torch.empty_like(q[85:]), pb.PL_F32)
            assert bool(torch.isnan(out).all()) == (bad != 0) and bool(torch.isnan(out).any()) == (bad != 0)
        caches.append(c)
    assert bool((caches[0].values(0, n).isnan() == torch.isnan(caches[0].scales[caches[0].table[0, :2].long(), 0])
                 .repeat_interleave(BLOCK, -1).permute(2, 0, 3, 1).reshape(2, -1, 2, 1)[:, :n]).all())
    if fmt == pb.PL_KV8_E4M3:  # no NaN among the codes of rows that exist
        code = caches[0].codes[caches[0].table[0, :2].long(), 0].permute(2, 0, 3, 1, 4).reshape(2, -1, kd)[:, :n]
        assert bool(((code & 127) != 127).all())
    for dtype in DTYPES:
        x = q.to(TORCH[dtype])
        out = caches[0].attend([0], [n], x, torch.empty_like(x), dtype)
        want, most, vmax = caches[1].reference([0], [n], x)
        assert bool(torch.isnan(out[80:]).all()) and not bool(torch.isnan(out[:80]).any())
        bound = attention_bound(dtype, head_dim, 128, most, vmax, want)
        assert bool(((out.double() - want).abs() <= bound)[:80].all())


@pytest.mark.parametrize("seqs,length", [(1, 20000), (3, 9001)])
def test_long_contexts_are_split(seqs, length):
    gen = generator(10)
    c = Cache(8, 1, 64, n_pages=seqs * 320, n_seqs=seqs, max_pages=320)
    c.fill(list(range(seqs)), [length - 777 * i for i in range(seqs)], gen)
    for count in (1, 5, 40):
        for dtype in (pb.PL_F32, pb.PL_BF16):
            attend_and_check(c, list(range(seqs)), [count] * seqs, dtype, gen)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("rise", [1, -1], ids=["rising", "falling"])
def test_outputs_leave_the_accumulator_several_times(fmt, head_dim, rise):
    """24 items of 188 tiles: on up to 160 SMs a block has at least 29 of
    their places, so most segments move O to its sums, every 4 tiles at
    head_dim 64 and every 8 at 128, three times or more.  Scores and V scales
    rise (or fall) all along, so the sums are rescaled as they are joined (or
    carry the output)."""
    gen = generator(35)
    c = Cache(16, 8, head_dim, fmt, n_pages=188, n_seqs=1, max_pages=188)
    c.fill([0], [12000], gen)
    pages = c.table[0].long()
    ramp = torch.linspace(-1, 1, 188 * 4, device="cuda").view(188, 1, 4) * rise
    c.scales[pages, 0, :, 0] *= 2.0 ** (2 * ramp)      # scores of +-0.25 to +-4 standard deviations
    c.scales[pages, 0, :, 1] *= 10.0 ** (4.5 * ramp - 1)  # values from 10^-5.5 to 10^3.5
    for dtype in (pb.PL_F32, pb.PL_F16):
        attend_and_check(c, [0], [300], dtype, gen)


def test_same_call_twice_gives_the_same_bits():
    gen = generator(11)
    c = Cache(32, 4, 64, n_pages=200, n_seqs=6, max_pages=64)
    lens = [1, 900, 2000, 17, 333, 1500]
    c.fill(list(range(6)), lens, gen)
    for counts in ([1] * 6, [1, 70, 200, 9, 33, 128]):
        q = randn(gen, sum(counts), 2048)
        a = c.attend(list(range(6)), counts, q, torch.empty_like(q), pb.PL_F32)
        b = c.attend(list(range(6)), counts, q, torch.empty_like(q), pb.PL_F32)
        assert torch.equal(a, b)


ROTATIONS = [dict(rope_dim=0), dict(rope_dim=10), dict(rope_dim=36), dict(rope_dim=48, base=500000.0), dict(),
             dict(rope_dim=32, scaling=pb.PL_ROPE_SCALE_YARN, factor=16.0, orig_len=64, low=1.0, high=32.0)]


@pytest.mark.parametrize("rotation", ROTATIONS, ids=["none", "10", "36", "48", "whole", "yarn32"])
@pytest.mark.parametrize("layout", [pb.PL_ROPE_LLAMA, pb.PL_ROPE_QWEN])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_attention_with_part_of_a_head_rotated(head_dim, layout, rotation):
    gen = generator(36)
    c = Cache(12, 4, head_dim, n_pages=32, n_seqs=3, max_pages=8, layout=layout, **rotation)
    c.fill([0, 1, 2], [300, 77, 512], gen)
    for dtype in DTYPES:
        attend_and_check(c, [2, 0, 1], [1, 1, 1], dtype, gen)
        attend_and_check(c, [2, 0, 1], [70, 3, 77], dtype, gen)


@pytest.mark.parametrize("rotation", ROTATIONS, ids=["none", "10", "36", "48", "whole", "yarn32"])
@pytest.mark.parametrize("layout", [pb.PL_ROPE_LLAMA, pb.PL_ROPE_QWEN])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("head_dim", [64, 128])
def test_decode_appends_as_append_does(head_dim, fmt, layout, rotation):
    """The decode step stores the codes and scales of pl_kv8_append_dev, at the
    start of a block, inside one and at its end, for rows that raise the
    scale, that do not, that are 0 and that are not finite; and attends them."""
    gen = generator(37)
    lens = [0, 1, 5, 14, 15, 16, 31, 63, 64, 100, 127, 9, 40, 70]  # before the step
    n, kd = len(lens), 4 * head_dim
    seqs = [int(i) for i in torch.randperm(n, generator=torch.Generator().manual_seed(2))]
    caches = [Cache(8, 4, head_dim, fmt, n_pages=48, n_seqs=n, max_pages=3, layout=layout, **rotation)
              for _ in range(2)]
    a, b = caches
    b.codes.copy_(a.codes)
    for c in caches:
        c.resize(seqs, lens)
    k, v = randn(gen, sum(lens), kd), randn(gen, sum(lens), kd)
    for c in caches:
        c.append(seqs, lens, k, v, pb.PL_F32)
    saved = [(c.codes.clone(), c.scales.clone()) for c in caches]
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales.view(torch.int32), b.scales.view(torch.int32))
    for c in caches:
        c.resize(seqs, [m + 1 for m in lens])
    for dtype in DTYPES:
        q, k, v = (randn(gen, n, w, dtype=TORCH[dtype]) for w in (2 * kd, kd, kd))
        k[1::3] *= 20          # raise the scales
        v[2::3] *= 20
        k[4], v[5] = 0, 0
        k[6, 3], k[7, kd - 1], v[8, head_dim], v[12, 5] = math.nan, math.inf, -math.inf, math.nan
        for c, (codes, scales) in zip(caches, saved):
            c.codes.copy_(codes)
            c.scales.copy_(scales)
        out = a.decode(seqs, q, k, v, torch.empty_like(q), dtype)
        b.append(seqs, [1] * n, k, v, dtype)
        assert torch.equal(a.codes, b.codes)
        assert torch.equal(a.scales.isnan(), b.scales.isnan())
        assert torch.equal(a.scales.nan_to_num(-1), b.scales.nan_to_num(-1))
        fine = [i for i in range(n) if i not in (6, 7, 8, 12)]
        t = torch.tensor(fine, device="cuda")
        want, most, vmax = a.reference([seqs[i] for i in fine], [1] * len(fine), q[t])
        assert bool(((out[t].double() - want).abs() <= attention_bound(dtype, head_dim, 128, most, vmax, want)).all())
        assert torch.equal(b.attend(seqs, [1] * n, q, torch.empty_like(q), dtype)[t], out[t])


# ------------------------------------------------------------------- pages
class Books:
    """The page operations in plain Python."""

    def __init__(self, n_pages, n_seqs):
        self.rows, self.pages, self.refs = [0] * n_seqs, [[] for _ in range(n_seqs)], [0] * n_pages
        self.data = list(range(n_pages))

    def resize(self, seqs, lens):
        rows, pages, refs = list(self.rows), [list(p) for p in self.pages], list(self.refs)
        for s, m in zip(seqs, lens):
            for p in pages[s][-(-m // PAGE):]:
                refs[p] -= 1
        shared = {}
        want = []
        for s, m in zip(seqs, lens):
            copy = False
            if m > rows[s] and rows[s] % PAGE:
                p = pages[s][rows[s] // PAGE]
                copy = refs[p] - shared.get(p, 0) > 1
                shared[p] = shared.get(p, 0) + 1
            want.append((copy, max(0, -(-m // PAGE) - -(-rows[s] // PAGE))))
        free = [p for p, r in enumerate(refs) if r == 0]
        if sum(c + n for c, n in want) > len(free):
            return False
        for (copy, more), s, m in zip(want, seqs, lens):
            del pages[s][-(-m // PAGE):]
            if copy:
                old, pages[s][-1] = pages[s][-1], free.pop(0)
                refs[old] -= 1
                refs[pages[s][-1]] = 1
                self.data[pages[s][-1]] = self.data[old]
            for _ in range(more):
                pages[s].append(free.pop(0))
                refs[pages[s][-1]] = 1
            rows[s] = m
        self.rows, self.pages, self.refs = rows, pages, refs
        return True

    def fork(self, src, dst):
        for a, b in zip(src, dst):
            for p in self.pages[b]:
                self.refs[p] -= 1
            for p in self.pages[a]:
                self.refs[p] += 1
            self.pages[b], self.rows[b] = list(self.pages[a]), self.rows[a]

    def compact(self):
        used = sum(r != 0 for r in self.refs)
        src = [p for p, r in enumerate(self.refs) if r and p >= used]
        dst = [p for p, r in enumerate(self.refs) if not r and p < used]
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.refs[b], self.refs[a], self.data[b] = self.refs[a], 0, self.data[a]
        self.pages = [[to.get(p, p) for p in s] for s in self.pages]


def check_books(c, b):
    assert c.lens.tolist() == b.rows
    assert c.refs.tolist() == b.refs
    width = c.table.shape[1]
    assert c.table.tolist() == [p + [-1] * (width - len(p)) for p in b.pages]
    used = [p for p, r in enumerate(b.refs) if r]
    for p in used:  # every page in use still holds its content
        assert bool((c.codes[p] == c.tag[b.data[p]]).all()) and bool((c.scales[p] == float(b.data[p])).all()), p


def tagged(n_pages, n_seqs, max_pages, **kw):
    """A cache whose page p holds the byte pattern of p."""
    c = Cache(4, 2, 64, n_pages=n_pages, n_seqs=n_seqs, max_pages=max_pages, **kw)
    c.tag = torch.randint(-128, 128, (n_pages,) + c.codes.shape[1:], device="cuda", generator=generator(12)).to(torch.int8)
    c.codes.copy_(c.tag)
    c.scales.copy_(torch.arange(n_pages, device="cuda").view(-1, 1, 1, 1, 1).expand_as(c.scales))
    return c, Books(n_pages, n_seqs)


@pytest.mark.parametrize("seed,layers", [(0, 1), (1, 3), (2, 2)])
def test_pages_against_plain_books(seed, layers):
    import random
    r = random.Random(seed)
    n_pages, n_seqs, max_pages = 26, 12, 9
    c, b = tagged(n_pages, n_seqs, max_pages, layers=layers)
    refused = 0
    for step in range(60):
        what = r.random()
        k = r.randint(1, n_seqs)
        seqs = r.sample(range(n_seqs), k)
        if what < 0.6:
            lens = [r.choice((0, b.rows[s], min(b.rows[s] + 1, 576), r.randint(0, 576), r.randint(0, 100))) for s in seqs]
            ok = b.resize(seqs, lens)
            refused += not ok
            c.resize(seqs, lens, pb.PL_OK if ok else pb.PL_ENOMEM)
        elif what < 0.85 and k >= 2:
            cut = r.randint(1, k - 1)
            src = [r.choice(seqs[:cut]) for _ in seqs[cut:]]
            b.fork(src, seqs[cut:])
            c.fork(src, seqs[cut:])
        else:
            b.compact()
            c.compact()
        check_books(c, b)
    assert refused > 0


def test_free_by_null_lengths():
    c, b = tagged(20, 3, 8)
    c.resize([0, 1], [200, 64])
    b.resize([0, 1], [200, 64])
    c.resize([1, 0])
    b.resize([1, 0], [0, 0])
    check_books(c, b)


def test_one_prompt_many_continuations():
    c, b = tagged(80, 40, 8, layers=2)
    for cache in (c, b):
        cache.resize([0], [130])
        cache.fork([0] * 39, list(range(1, 40)))
    check_books(c, b)
    for cache in (c, b):  # slot 0 too: the last of the list keeps the shared page
        cache.resize(list(range(39, -1, -1)), [131] * 40)
    check_books(c, b)
    assert sum(c.refs.tolist()) == 40 * 3 and c.refs.max() == 40


def test_copy_pages():
    c, _ = tagged(40, 2, 4)
    a, b = i32([3, 9, 9, 0]), i32([39, 1, 20, 38])
    c.c.copy_dev(4, a.data_ptr(), b.data_ptr(), stream())
    assert c.c.status(stream()) == pb.PL_OK
    want = list(range(40))
    want[39], want[1], want[20], want[38] = 3, 9, 9, 0
    for p in range(40):
        assert bool((c.codes[p] == c.tag[want[p]]).all()) and bool((c.scales[p] == float(want[p])).all())
    for src, dst in (([1, 2], [5, 5]), ([1, 5], [5, 6]), ([1], [40]), ([-1], [2])):
        x, y = i32(src), i32(dst)
        before = c.codes.clone()
        c.c.copy_dev(len(src), x.data_ptr(), y.data_ptr(), stream())
        assert c.c.status(stream()) == pb.PL_EARG
        assert torch.equal(c.codes, before)


def test_large_pools():
    """More pages and cells than one pass of the plan's block."""
    c = Cache(1, 1, 64, n_pages=5000, n_seqs=300, max_pages=700)
    b = Books(5000, 300)
    lens = [(i * 37) % 900 + (40000 if i == 7 else 0) for i in range(300)]
    assert b.resize(list(range(300)), lens)
    c.resize(list(range(300)), lens)
    half = list(range(0, 300, 2))
    b.resize(half, [0] * 150)
    c.resize(half)
    b.compact()
    c.compact()
    assert c.lens.tolist() == b.rows and c.refs.tolist() == b.refs
    assert [[p for p in row if p >= 0] for row in c.table.tolist()] == b.pages


@pytest.mark.parametrize("n_seqs,max_pages", [(1024, 2 ** 21), (1024, 2 ** 22), (256, 2 ** 23 + 1)])
def test_more_pages_than_31_bits_count(n_seqs, max_pages):
    """Entries that want 2^31 pages, 2^32 and 2^31 + 256 between them: too
    many for the pool, which keeps everything.  (Nothing is written to the
    table, 8 to 17 GB, so it is left as it was allocated.)"""
    geometry = dict(n_layers=1, n_heads=1, n_kv_heads=1, head_dim=64, n_pages=300, n_seqs=n_seqs, max_pages=max_pages)
    codes = torch.zeros(300 * 2 * 64 * 64, dtype=torch.int8, device="cuda")
    scales = torch.zeros(300 * 8, device="cuda")
    table = torch.empty(n_seqs * max_pages, dtype=torch.int32, device="cuda")
    lens, refs = torch.zeros(n_seqs, dtype=torch.int32, device="cuda"), torch.zeros(300, dtype=torch.int32, device="cuda")
    work = torch.zeros(pb.kv8_work_bytes(**geometry), dtype=torch.uint8, device="cuda")
    c = pb.Kv8Cache(**geometry, codes=codes.data_ptr(), scales=scales.data_ptr(), table=table.data_ptr(),
                    lens=lens.data_ptr(), refs=refs.data_ptr(), work=work.data_ptr(), work_bytes=work.numel())
    seqs, want = i32(list(range(n_seqs))), i32([max_pages * PAGE] * n_seqs)
    c.resize_dev(n_seqs, seqs.data_ptr(), want.data_ptr(), stream())
    assert c.status(stream()) == pb.PL_ENOMEM
    assert not bool(lens.any()) and not bool(refs.any())
    # and the pool still serves what fits
    want.fill_(0)
    want[:300] = 64 if n_seqs >= 300 else 1
    c.resize_dev(n_seqs, seqs.data_ptr(), want.data_ptr(), stream())
    assert c.status(stream()) == pb.PL_OK
    assert torch.equal(lens, want) and int(refs.sum()) == min(n_seqs, 300)
    del table
    torch.cuda.empty_cache()


# --------------------------------------------------------------- refusals
def test_bad_entries_are_reported_and_left_undone():
    gen = generator(13)
    c = Cache(4, 2, 64, n_seqs=3)
    c.fill([0, 1, 2], [40, 50, 60], gen)
    books = [x.clone() for x in (c.table, c.lens, c.refs, c.codes)]

    def same():
        return all(torch.equal(x, y) for x, y in zip(books, (c.table, c.lens, c.refs, c.codes)))

    c.resize([0, 3], [64, 64], pb.PL_EARG)
    c.resize([0, 0], [64, 70], pb.PL_EARG)
    c.resize([0, 1], [64, -1], pb.PL_EARG)
    c.resize([0, 1], [64, 8 * 64 + 1], pb.PL_EARG)
    c.resize([0], [8 * 64], pb.PL_OK)
    c.resize([0], [40], pb.PL_OK)
    c.fork([0, 1], [2, 2], pb.PL_EARG)
    c.fork([0], [0], pb.PL_EARG)
    c.fork([0, 1], [1, 2], pb.PL_EARG)
    c.fork([0, 5], [1, 2], pb.PL_EARG)
    assert same()
    # attention: a slot out of range, tokens past `total`; the other entry is computed
    q = randn(gen, 4, 256)
    for seqs, st in (([-1, 1], [0, 1, 2]), ([7, 1], [0, 1, 2]), ([0, 1], [-1, 1, 2]), ([0, 1], [3, 2, 3])):
        out = torch.full_like(q, 5.0)
        a, s = i32(seqs), i32(st)
        c.c.attend_dev(0, 2, a.data_ptr(), s.data_ptr(), 3, 2, pb.PL_F32, q.data_ptr(), 256, out.data_ptr(), 256, stream())
        assert c.c.status(stream()) == pb.PL_EARG
        assert c.c.status(stream()) == pb.PL_OK
        got = out[st[1]:st[2]].double()
        want, most, vmax = c.reference([1], [st[2] - st[1]], q[st[1]:st[2]])
        assert bool(((got - want).abs() <= attention_bound(pb.PL_F32, 64, 64, most, vmax, want)).all())
    # a table entry that names no page
    c.table[1, 0] = 1000
    out = torch.full_like(q, 5.0)
    a = i32([1])
    for count in (1, 2):
        st = i32([0, count])
        c.c.attend_dev(0, 1, a.data_ptr(), st.data_ptr(), count, count, pb.PL_F32, q.data_ptr(), 256, out.data_ptr(), 256,
                       stream())
        assert c.c.status(stream()) == pb.PL_EARG
    c.c.append_dev(0, 1, a.data_ptr(), None, 1, 1, pb.PL_F32, q.data_ptr(), 256, q.data_ptr(), 256, stream())
    assert c.c.status(stream()) == pb.PL_EARG
    assert torch.equal(c.codes, books[3])


def test_allocated_by_the_module(monkeypatch):
    with pb.Kv8Cache(2, 8, 2, n_pages=10, n_seqs=2, max_pages=4) as c:
        s, n = i32([1]), i32([70])
        c.resize_dev(1, s.data_ptr(), n.data_ptr(), stream())
        k = randn(generator(14), 70, 128)
        st = i32([0, 70])
        c.append_dev(1, 1, s.data_ptr(), st.data_ptr(), 70, 70, pb.PL_F32, k.data_ptr(), 128, k.data_ptr(), 128, stream())
        out, zero = torch.empty(70, 128, device="cuda"), i32([0])
        c.read_dev(1, 1, s.data_ptr(), zero.data_ptr(), st.data_ptr(), 70, 70, pb.PL_F32, out.data_ptr(), 128,
                   out.data_ptr(), 128, stream())
        assert c.status(stream()) == pb.PL_OK
        # without a rotation given, rows are stored as they come: within half a step of the block's largest
        assert float((out - k).abs().max()) <= float(k.abs().max()) / 127 * 0.51
        with pytest.raises(pb.PlAttnError) as e:
            c.append_dev(2, 1, s.data_ptr(), None, 1, 1, pb.PL_F32, k.data_ptr(), 128, k.data_ptr(), 128, stream())
        assert e.value.rc == pb.PL_EARG
    with pytest.raises(pb.PlAttnError) as e:
        pb.Kv8Cache(1, 8, 2, n_pages=4, n_seqs=2, max_pages=4, device=63)
    assert e.value.rc == pb.PL_EDEVICE


# ------------------------------------------------------------ used together
@pytest.mark.parametrize("fmt,dtype,head_dim", [(pb.PL_KV8_INT8, pb.PL_F32, 64), (pb.PL_KV8_E4M3, pb.PL_BF16, 128),
                                                (pb.PL_KV8_INT8, pb.PL_F16, 128)])
def test_prompt_fork_decode_and_compact_together(fmt, dtype, head_dim):
    """A prompt in two chunks, three continuations of it, decode steps of
    all with one ending on the way, over two layers; after each call the
    output is that of the rows stored so far."""
    gen = generator(15)
    heads, kvh = 8, 2
    c = Cache(heads, kvh, head_dim, fmt, n_pages=40, n_seqs=6, max_pages=6, layers=2, layout=pb.PL_ROPE_QWEN,
              base=500000.0, scaling=pb.PL_ROPE_SCALE_LLAMA3, factor=8.0, orig_len=64)
    kd = kvh * head_dim
    plain = {}                                       # slot -> per layer [2][rows][kv heads][hd], unquantised

    def step(seqs, counts, one=False):
        lens = [int(c.lens[s]) + n for s, n in zip(seqs, counts)]
        c.resize(seqs, lens)
        for layer in range(2):
            q, k, v = (randn(gen, sum(counts), w, dtype=TORCH[dtype]) for w in (heads * head_dim, kd, kd))
            out = torch.empty_like(q)
            if one:
                c.decode(seqs, q, k, v, out, dtype, layer)
            else:
                c.append(seqs, counts, k, v, dtype, layer)
                c.attend(seqs, counts, q, out, dtype, layer)
            want, most, vmax = c.reference(seqs, counts, q, layer)
            assert bool(((out.double() - want).abs() <= attention_bound(dtype, head_dim, max(lens), most, vmax, want)).all())
            t = 0
            for s, n, m in zip(seqs, counts, lens):
                kr = rotate(k[t:t + n].view(n, kvh, head_dim), torch.arange(m - n, m, device="cuda"), c.freq, c.gain,
                            c.layout)
                new = torch.stack((kr, v[t:t + n].double().view(n, kvh, head_dim)))
                had = plain.get((s, layer), new[:, :0])
                plain[s, layer] = torch.cat((had, new), 1)
                t += n

    step([0], [70])
    step([0], [58])
    step([3], [9])
    c.fork([0, 0, 0], [1, 2, 4])
    for s in (1, 2, 4):
        for layer in range(2):
            plain[s, layer] = plain[0, layer]
    for i in range(20):
        step([4, 0, 3, 1, 2] if i < 9 else [4, 0, 2], [1] * (5 if i < 9 else 3), one=True)
        if i == 8:
            c.resize([3, 1])
            c.compact()
            used = int((c.refs > 0).sum())
            assert bool((c.refs[:used] > 0).all())
    # what is stored is within the steps of its format of what was appended:
    # half a step for the rounding, and half a step more for each of up to
    # 15 later rows that raised the scale of its block
    for s in (0, 2, 4):
        for layer in range(2):
            got, x = c.values(s, plain[s, layer].shape[1], layer), plain[s, layer]
            top = float(x.abs().max())
            limit = 8 * top / 127 if fmt == pb.PL_KV8_INT8 else 8 * torch.maximum(x.abs() / 16, torch.full_like(x, top / 448 / 1024)) * 1.5
            assert bool(((got - x).abs() <= limit).all())


def test_captured_step_replayed():
    """A step (grow, append, attend) captured in a graph on another stream
    and replayed: every replay appends the next token."""
    gen = generator(16)
    c = Cache(8, 2, 64, n_pages=32, n_seqs=3, max_pages=8)
    c.fill([0, 1, 2], [60, 1, 127], gen)
    lens, seqs = i32([60, 1, 127]), i32([0, 1, 2])
    q, k, v = randn(gen, 3, 512), randn(gen, 3, 128), randn(gen, 3, 128)
    out = torch.zeros_like(q)

    def one():
        lens.add_(1)
        c.c.resize_dev(3, seqs.data_ptr(), lens.data_ptr(), stream())
        c.c.decode_dev(0, 3, seqs.data_ptr(), pb.PL_F32, q.data_ptr(), 512, k.data_ptr(), 128, v.data_ptr(), 128,
                       out.data_ptr(), 512, stream())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one()
    for i in range(6):
        q.copy_(randn(gen, 3, 512))
        k.copy_(randn(gen, 3, 128))
        v.copy_(randn(gen, 3, 128))
        graph.replay()
        assert c.c.status(stream()) == pb.PL_OK
        assert c.lens.tolist() == [60 + i + 2, 1 + i + 2, 127 + i + 2]
        want, most, vmax = c.reference([0, 1, 2], [1, 1, 1], q)
        assert bool(((out.double() - want).abs() <= attention_bound(pb.PL_F32, 64, 140, most, vmax, want)).all())
    del graph


# ---------------------------------------------------------- less usual calls
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("split", [1, 7, 8, 9, 15])
def test_append_joins_a_block_of_wide_heads(fmt, split):
    """Two warps share a block of 16 rows of 128 elements: the scale and the
    kept rows cross between them, whichever of them holds the new rows."""
    gen = generator(21)
    c = Cache(4, 2, 128, fmt)
    k, v = randn(gen, 16, 256), randn(gen, 16, 256)
    k[split:] *= 40
    v[15] *= 40
    c.resize([0], [split])
    c.append([0], [split], k[:split], v[:split], pb.PL_F32)
    kr = rotate(k.double().reshape(16, 2, 128), torch.arange(16, device="cuda"), c.freq, c.gain, c.layout)
    vr = v.double().reshape(16, 2, 128)
    old = c.values(0, split).clone()
    page = int(c.table[0, 0])
    old_s = c.scales[page, 0, :, :, 0].double().clone()
    for kv, x in ((0, kr), (1, vr)):
        check_rows(c, 0, 0, split, x[:split], kv)
    c.resize([0], [16])
    c.append([0], [16 - split], k[split:], v[split:], pb.PL_F32)
    s = c.scales[page, 0, :, :, 0].double()
    assert bool((s > old_s).all())
    # the new rows to half a step; the kept ones to half a step of the new scale from what they were,
    # the ratio of the scales, its product and the code's value rounded once each
    got = c.values(0, 16)
    for kv, x in ((0, kr), (1, vr)):
        check_rows(c, 0, split, 16, x[split:], kv)
        step = s[:, kv][:, None]
        half = 0.5 * step if fmt == pb.PL_KV8_INT8 else torch.maximum(old[kv].abs() / 16, step * 2.0 ** -10)
        assert bool(((got[kv, :split] - old[kv]).abs() <= half * (1 + 2.0 ** -15)).all())


@pytest.mark.parametrize("row", [0, 7, 8, 15])
def test_append_of_a_nonfinite_wide_row(row):
    c = Cache(2, 2, 128)
    c.resize([0], [16])
    k, v = torch.zeros(16, 256, device="cuda"), torch.zeros(16, 256, device="cuda")
    k[row, 5], v[row, 200] = -math.inf, math.nan
    c.append([0], [16], k, v, pb.PL_F32)
    got = c.values(0, 16)
    assert bool(torch.isnan(got[0, :, 0]).all()) and bool((got[0, :, 1] == 0).all())
    assert bool(torch.isnan(got[1, :, 1]).all()) and bool((got[1, :, 0] == 0).all())


def test_attention_may_name_a_slot_twice():
    gen = generator(22)
    c = Cache(8, 2, 64, n_pages=64, n_seqs=3, max_pages=8)
    c.fill([0, 1, 2], [300, 77, 512], gen)
    for seqs, counts in (([2, 0, 2, 2], [1] * 4), ([0, 0, 1, 0], [40, 40, 3, 7])):
        attend_and_check(c, seqs, counts, pb.PL_F32, gen)


def test_status_on_a_stream_that_waits_for_no_other():
    """An error after one that was read is not lost to the clearing of it."""
    c = Cache(4, 2, 64, n_seqs=2)
    bad, n = i32([5]), i32([3])
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        for _ in range(50):
            c.c.resize_dev(1, bad.data_ptr(), n.data_ptr(), stream())
            assert c.c.status(stream()) == pb.PL_EARG
        assert c.c.status(stream()) == pb.PL_OK
    torch.cuda.synchronize()


def test_waits_that_run_out_are_reported():
    """A block's scheduler stays four segments ahead of the others, and waits
    for a segment to end before it names a fifth: here, with seven segments
    of 1024 tiles a block, for 0.28 ms at least (a tile's 8192 exponentials at
    16 a clock take 0.27 us).  With a limit of 0.1 ms, after which a wait ends
    within 0.04 ms, that runs out: the call says PL_ETIMEOUT, and the next one,
    with the limit back, is right again."""
    gen = generator(33)
    c = Cache(16, 2, 64, n_pages=1024, n_seqs=1, max_pages=1024)
    c.fill([0], [65536], gen)
    n = 512
    q = randn(gen, 2 * n, 1024)
    seqs, counts = [0] * n, [2] * n
    want = c.attend(seqs, counts, q, torch.empty_like(q), pb.PL_F32)
    for t in (0, 2 * n - 2):
        exact, most, vmax = c.reference([0], [2], q[t:t + 2])
        assert bool(((want[t:t + 2].double() - exact).abs() <=
                     attention_bound(pb.PL_F32, 64, 65536, most, vmax, exact)).all())
    a, st = i32(seqs), i32(starts(counts))
    with pb.Attn(1, 8, 2, 64) as at:
        for _ in range(2):
            at.set_wait_limit(1e-4)
            out = torch.empty_like(q)
            c.c.attend_dev(0, n, a.data_ptr(), st.data_ptr(), 2 * n, 2, pb.PL_F32, q.data_ptr(), 1024,
                           out.data_ptr(), 1024, stream())
            rc = c.c.status(stream())
            at.set_wait_limit(2.0)
            assert rc == pb.PL_ETIMEOUT
            assert c.c.status(stream()) == pb.PL_OK
            assert torch.equal(c.attend(seqs, counts, q, out, pb.PL_F32), want)


def test_wait_limit_ends_with_its_context():
    """The call of the test above, after a context that had set 0.1 ms."""
    gen = generator(34)
    c = Cache(16, 2, 64, n_pages=1024, n_seqs=1, max_pages=1024)
    c.fill([0], [65536], gen)
    q = randn(gen, 1024, 1024)
    with pb.Attn(1, 8, 2, 64) as at:
        at.set_wait_limit(1e-4)
    c.attend([0] * 512, [2] * 512, q, torch.empty_like(q), pb.PL_F32)  # checks the status


def test_two_caches_on_two_streams():
    """Caches are independent: their calls may overlap."""
    gen = generator(23)
    caches = [Cache(8, 2, hd, n_pages=130, n_seqs=2, max_pages=64) for hd in (64, 128)]
    runs = []
    for c in caches:
        c.fill([0, 1], [3000, 4000], gen)
        q = randn(gen, 130, 8 * c.head_dim)
        runs.append((c, q, [torch.empty_like(q) for _ in range(2)], i32([0, 1]), i32([0, 65, 130]), torch.cuda.Stream()))
    for alone in (True, False):
        torch.cuda.synchronize()
        for _ in range(1 if alone else 8):
            for c, q, out, s, st, on in runs:
                c.c.attend_dev(0, 2, s.data_ptr(), st.data_ptr(), 130, 65, pb.PL_F32, q.data_ptr(), q.stride(0),
                               out[alone].data_ptr(), q.stride(0), on.cuda_stream)
                if alone:
                    torch.cuda.synchronize()
    for c, _, out, _, _, on in runs:
        assert c.c.status(on.cuda_stream) == pb.PL_OK
        assert torch.equal(out[0], out[1])


@pytest.mark.parametrize("page", [-1, 1000])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_decode_without_a_page_writes_nothing(page, head_dim):
    """A new row whose page is missing is not written anywhere; another entry's step is made."""
    gen = generator(26)
    c = Cache(4, 2, head_dim, n_seqs=3)
    c.fill([0, 1, 2], [40, 129, 64], gen)
    at = int(c.table[2, 0])
    c.table[1, 2] = page
    codes, scales = c.codes.clone(), c.scales.clone()
    q, k, v = randn(gen, 2, 4 * head_dim), randn(gen, 2, 2 * head_dim), randn(gen, 2, 2 * head_dim)
    out, s = torch.empty_like(q), i32([1, 2])
    c.c.decode_dev(0, 2, s.data_ptr(), pb.PL_F32, q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0),
                   v.data_ptr(), v.stride(0), out.data_ptr(), out.stride(0), stream())
    assert c.c.status(stream()) == pb.PL_EARG
    changed = (c.codes != codes).flatten(1).any(1) | (c.scales.nan_to_num(9) != scales.nan_to_num(9)).flatten(1).any(1)
    assert changed.nonzero().flatten().tolist() == [at]
    want, most, vmax = c.reference([2], [1], q[1:])
    assert bool(((out[1:].double() - want).abs() <= attention_bound(pb.PL_F32, head_dim, 64, most, vmax, want)).all())


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("counts", [[1, 1], [200, 3]])
def test_fp16_is_off_by_its_output_alone(head_dim, counts):
    """FP16 activations are carried as FP32 ones are, and the output is
    rounded once: half a step of 2^-11, or half a subnormal's 2^-25."""
    gen = generator(25)
    c = Cache(8, 2, head_dim, n_pages=40, n_seqs=2, max_pages=20)
    c.fill([0, 1], [700, 1200], gen)
    q = randn(gen, sum(counts), 8 * head_dim, dtype=torch.float16)
    out = c.attend([0, 1], counts, q, torch.empty_like(q), pb.PL_F16)
    want, most, vmax = c.reference([0, 1], counts, q)
    bound = attention_bound(pb.PL_F32, head_dim, 1200, most, vmax, want) + want.abs() * 2.0 ** -11 + 2.0 ** -25
    assert bool(((out.double() - want).abs() <= bound).all())


def test_many_entries_of_one_call():
    """As many entries as a call takes, most of them short and some empty."""
    gen = generator(24)
    n = 1024
    c = Cache(2, 1, 64, n_pages=1500, n_seqs=n, max_pages=2)
    lens = [(7 * i) % 97 for i in range(n)]
    c.fill(list(range(n)), lens, gen)
    attend_and_check(c, list(range(n)), [1] * n, pb.PL_BF16, gen)
    attend_and_check(c, list(range(n)), [min(m, (3 * i) % 5) for i, m in enumerate(lens)], pb.PL_BF16, gen)
    c.resize(list(range(n)))
    assert int(c.refs.abs().sum()) == 0


def test_the_integration_guide_runs():
    """The Python example of the guide, as written."""
    import pathlib
    import re

    text = (pathlib.Path(__file__).resolve().parent.parent / "INTEGRATION.md").read_text()
    blocks = [b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "Kv8Cache" in b]
    assert len(blocks) == 1
    scope = {}
    exec(blocks[0], scope)
    # one row attends itself: the output is v, a head for each group of 8, to int8
    want = scope["v"].view(2, 4, 1, 64).expand(2, 4, 8, 64).reshape(2, 2048)
    assert float((scope["out"] - want).abs().max()) <= float(want.abs().max()) / 127 * 0.51
