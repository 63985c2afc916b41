"""The K/V cache in 8 bits: writes bit for bit, attention over what the codes and scales stand for against 64 bits.

Tolerance of the attention.  u: half a unit of the last place of the output's type.  With S_t = sum_d scale |q_d k_td| (at most S) and n
tokens, the fp32 score of a token is off by at most (D + 2) 2^-24 S, its weight by that (relative, in the exponent) and by 2^-11 for a
rounding of it to fp16, a sum of n weights or products by n 2^-24: with size = sum_t p_t |v_t|, all of it twice over (numerator and
denominator)
    |x - y| <= u |y| + (2 (D + 2) 2^-24 S + 2 n 2^-24 + w) size,   w = 2^-11, fp32: 2^-22 (the exponential),
and 2^-25 for fp16 outputs below the normal range.  A weight times its block's value scale is kept so that the largest is 2^7 at least:
one below 2^-14, fp16's normal range, is off by 2^-25 instead, so the output by
    2^-25 2^-7 max_t (p_t s_t) sum_t |code_t|
more, which shows where the tokens that have the weight have next to nothing in a dimension."""
import os
import subprocess
import sys

import pytest
import torch

from apt_serve_b200 import attention as A
from apt_serve_b200 import ops
from apt_serve_b200.cache_engine import CacheEngine
from apt_serve_b200.layers import OPTAttention
from apt_serve_b200.metadata import BlockPool  # noqa: F401

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
F32, F, B = torch.float32, torch.float16, torch.bfloat16
U = {F32: 2.0 ** -24, F: 2.0 ** -11, B: 2.0 ** -8}
DEV = "cuda"


# ---- the definition ----------------------------------------------------------------------
def needed(top):
    """The smallest power of two s >= 2^-118 with top <= 448 s."""
    m, e = torch.frexp(top.double().clamp_min(2.0 ** -120) / 448)   # of nothing but zeros: the least
    return torch.ldexp(torch.ones_like(m), (e - (m == 0.5).int()).clamp_min(-118))


def write_reference(codes, scales, rows, slots, bs):
    """One plane on the CPU: codes uint8 [NB, BS, H, D], scales [NB, H], rows [T, H, D]; changed in place."""
    by_block = {}
    for t, s in enumerate(slots):
        if 0 <= s < codes.shape[0] * bs:
            by_block.setdefault(s // bs, {})[s % bs] = t   # the later of two rows for a slot stays
    for b, some in by_block.items():
        x = rows[[some[o] for o in some]].double()
        fine = torch.isfinite(x)
        need = needed(torch.where(fine, x.abs(), torch.zeros_like(x)).amax(dim=(0, 2)))
        anew = 0 in some
        old = scales[b].double()
        new = need if anew else torch.maximum(old, need)
        if not anew:
            moved = (new != old)[None, :, None]
            kept = (codes[b].view(E4M3).double() * (old / new)[None, :, None]).float().to(E4M3).view(torch.uint8)
            codes[b] = torch.where(moved, kept, codes[b])
        y = torch.where(fine, x / new[None, :, None], torch.full_like(x, float("nan"))).float().to(E4M3).view(torch.uint8)
        for i, o in enumerate(some):
            codes[b, o] = y[i]
        scales[b] = new.float()


def same_codes(a, b):
    a, b = a.cpu().view(torch.uint8), b.cpu().view(torch.uint8)
    nan = (a & 0x7f == 0x7f) & (b & 0x7f == 0x7f)
    return bool(((a == b) | nan).all())


def attention_reference(q, k8, v8, ks, vs, tables, starts, lens, scale):
    """[T, H, D] outputs in 64 bits, sum p |v|, S and n of the rows, what small weights add; NaN where a row belongs to no request."""
    t, h, d = q.shape
    bs, most = k8.shape[1], tables.shape[1] * k8.shape[1]
    out, size, least = (torch.full((t, h, d), float("nan"), dtype=torch.double, device=DEV) for _ in range(3))
    score, count = torch.zeros(t, h, 1, dtype=torch.double, device=DEV), torch.zeros(t, 1, 1, dtype=torch.double, device=DEV)
    for r, n in enumerate(lens):
        a, b = starts[r], starts[r + 1]
        n = max(0, min(n, most))
        ids = tables[r, :-(-n // bs)].long()
        k, v = ((c.view(torch.uint8)[ids].view(E4M3).double() * s[ids].double()[:, None, :, None]).flatten(0, 1)[:n]
                for c, s in ((k8, ks), (v8, vs)))
        codes = v8.view(torch.uint8)[ids].view(E4M3).double().abs().flatten(0, 1)[:n]
        steps = vs[ids].double().repeat_interleave(bs, 0)[:n]
        for i in range(a, b):
            keys = n - (b - 1 - i)
            if keys <= 0:
                out[i], size[i], least[i] = 0.0, 0.0, 0.0
                continue
            each = q[i].double()[None] * k[:keys] * scale
            p = torch.softmax(each.sum(2), dim=0)
            out[i] = torch.einsum("kh,khd->hd", p, v[:keys])
            size[i] = torch.einsum("kh,khd->hd", p, v[:keys].abs())
            least[i] = 2.0 ** -32 * (p * steps[:keys]).amax(0)[:, None] * codes[:keys].sum(0)
            score[i, :, 0] = each.abs().sum(2).amax(0)
            count[i] = keys
    return out, size, score, count, least


def check(got, ref, dtype):
    out, size, score, count, least = ref
    t, h, d = out.shape
    got = got.double().view(t, h, d)
    w = 2.0 ** -22 if dtype == F32 else 2.0 ** -11
    bound = U[dtype] * out.abs() + (2 * (d + 2) * 2.0 ** -24 * score + 2 * count * 2.0 ** -24 + w) * size
    bound = bound + (2.0 ** -25 if dtype == F else 0.0) + (0.0 if dtype == F32 else least) + 1e-300
    bad = ~((got - out).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist(), float(((got - out).abs() / bound).max()))


# ---- inputs -----------------------------------------------------------------------------
def make_cache(nb, bs, h, d, seed=0, pad=0, spread=True, storage=E4M3):
    """Caches with codes of normal numbers and scales that are no powers of two, `pad` more bytes from block to block."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    flat = torch.randn(2, nb, bs * h * d + pad, generator=g, device=DEV).mul_(40).clamp_(-448, 448).to(E4M3).view(torch.uint8)
    cache = flat[:, :, :bs * h * d].view(2, nb, bs, h, d)
    scales = torch.rand(2, nb, h, generator=g, device=DEV).add_(0.5).div_(40)
    if spread:
        scales *= torch.exp2(torch.randint(-3, 4, (2, nb, h), generator=g, device=DEV).float())
    return cache.view(storage), scales


def make_tables(lens, bs, nb, seed=0, width=None):
    g = torch.Generator().manual_seed(seed)
    per = [-(-max(0, n) // bs) for n in lens]
    assert sum(per) <= nb
    ids = torch.randperm(nb, generator=g)[:sum(per)].tolist()
    tables = torch.full((len(lens), max(per + [1]) if width is None else width), nb + 7, dtype=torch.int32)   # never to be read
    at = 0
    for r, p in enumerate(per):
        tables[r, :p] = torch.tensor(ids[at:at + p], dtype=torch.int32)
        at += p
    return tables.to(DEV)


def spoil_behind(cache, tables, lens, bs):
    """NaN codes in the rows behind each request's last token."""
    raw = cache.view(torch.uint8)
    for r, n in enumerate(lens):
        if n > 0 and n % bs:
            raw[:, int(tables[r, n // bs]), n % bs:] = 0x7f


def query(t, h, d, dtype, seed=0, spread=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed + 100)
    return torch.randn(t, 3, h, d, generator=g, device=DEV).mul_(spread).to(dtype).view(t, 3 * h * d)[:, :h * d]   # of a projection


# ---- writes -----------------------------------------------------------------------------
def rows_of(t, h, d, dtype, seed, magnitude=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed + 50)
    x = torch.randn(t, 3, h, d, generator=g, device=DEV) * torch.exp2(torch.randint(-6, 7, (t, 3, h, 1), generator=g, device=DEV).float())
    x = (x * magnitude).to(dtype).view(t, 3 * h * d)
    return x[:, h * d:2 * h * d].view(t, h, d), x[:, 2 * h * d:].view(t, h, d)


def check_write(cache, scales, key, value, slots, bs):
    want = [(cache[p].cpu().view(torch.uint8).clone(), scales[p].cpu().clone()) for p in (0, 1)]
    for p, rows in ((0, key), (1, value)):
        write_reference(*want[p], rows.cpu(), slots, bs)
    for _ in range(2):   # a second time changes nothing
        ops.reshape_and_cache_flash(key, value, cache[0], cache[1], torch.tensor(slots, device=DEV, dtype=torch.int64), "fp8", scales[0], scales[1])
        for p in (0, 1):
            assert torch.equal(scales[p].cpu(), want[p][1])
            assert same_codes(cache[p].reshape(want[p][0].shape), want[p][0])


@pytest.mark.parametrize("dtype", [F32, F, B])
@pytest.mark.parametrize("h,d,bs", [(3, 64, 16), (2, 128, 16), (5, 32, 32), (1, 256, 48), (9, 128, 32)])
def test_write_of_prompts_and_tokens(h, d, bs, dtype):
    """Whole prompts, single tokens behind and at the start of blocks, rows in any order, negative slots, a slot twice, zeros."""
    cache, scales = make_cache(24, bs, h, d, seed=h + d)
    slots = list(range(2 * bs, 5 * bs - 3)) + [-1, 7 * bs + 3, 9 * bs, 11 * bs + bs - 1] + list(range(13 * bs, 13 * bs + 2))
    slots += [15 * bs + 5, 16 * bs, 15 * bs + 2, -1, 16 * bs + 1, 15 * bs + 5] + list(range(20 * bs + 7, 22 * bs))[::-1] + [0]
    key, value = rows_of(len(slots), h, d, dtype, seed=d)
    key[3] = 0
    value[len(slots) - 1] = 0   # a block of nothing but zeros: the least scale
    check_write(cache, scales, key, value, slots, bs)


@pytest.mark.parametrize("dtype", [F32, F, B])
def test_write_of_special_values(dtype):
    bs, h, d = 16, 2, 64
    cache, scales = make_cache(8, bs, h, d, seed=5)
    slots = list(range(0, 16)) + [16 + 9, 32 + 4, 48, 64 + 3, 80 + 1]
    key, value = rows_of(len(slots), h, d, dtype, seed=1)
    key[2, 0, 5], key[3, 1, 6], value[4, 0, 7] = float("nan"), float("inf"), -float("inf")
    key[16] = float("nan")                           # nothing finite: the scale stays, the row is NaN
    value[17] = torch.finfo(dtype).max
    key[18, 0] = torch.finfo(dtype).tiny / 4         # a subnormal number
    key[19] *= 2.0 ** -12                            # far below what the block holds
    value[19, 0, :] = 448 * 2.0 ** -3                # the largest number that a scale takes, and the next one
    value[19, 1, :] = 449 * 2.0 ** -3 if dtype != B else 450 * 2.0 ** -3
    scales[1, 5] = 0.0                               # a block that nothing was written to
    check_write(cache, scales, key, value, slots, bs)


def test_write_of_rows_that_are_not_aligned():
    bs, h, d = 16, 3, 64
    for dtype in (F, F32):
        cache, scales = make_cache(6, bs, h, d, seed=2, pad=16)
        wide = torch.randn(20, 2 * h * d + 3, device=DEV).to(dtype)
        key, value = wide[:, 1:1 + h * d].unflatten(1, (h, d)), wide[:, h * d + 2:2 * h * d + 2].unflatten(1, (h, d))
        check_write(cache, scales, key, value, list(range(16, 30)) + [33, 34, 35, 64, 65, 95], bs)


def test_write_of_a_single_row_with_any_stride():
    cache, scales = make_cache(4, 16, 2, 64, seed=3, storage=torch.uint8)
    key, value = rows_of(1, 2, 64, F, seed=4)
    check_write(cache, scales, key, value, [18], 16)


def test_write_many_rows_in_any_order():
    """More rows than a single CTA looks through, in and out of order, beside blocks that are left alone."""
    bs, h, d, nb = 16, 2, 64, 700
    g = torch.Generator().manual_seed(9)
    cache, scales = make_cache(nb, bs, h, d, seed=6)
    every = torch.randperm(nb * bs, generator=g)[:5000].tolist()
    runs = [s for b in range(0, 300) for s in range(b * bs, b * bs + bs)]
    for slots in (every, runs, every[:1500] + runs[:3000]):
        key, value = rows_of(len(slots), h, d, B, seed=7)
        check_write(cache.clone(), scales.clone(), key, value, slots, bs)


def test_write_slots_past_the_cache_are_reported():
    A.raise_on_device_status()
    cache, scales = make_cache(4, 16, 2, 64, seed=3)
    key, value = rows_of(4, 2, 64, F, seed=4)
    check_write(cache, scales, key, value, [5, 4 * 16, 2 ** 40, 6], 16)
    with pytest.raises(RuntimeError, match="outside its tensors"):
        A.raise_on_device_status()
    A.raise_on_device_status()


def test_write_of_nothing():
    cache, scales = make_cache(4, 16, 2, 64, seed=3)
    before = cache.view(torch.uint8).clone()
    key, value = rows_of(3, 2, 64, F, seed=4)
    ops.reshape_and_cache_flash(key[:0], value[:0], cache[0], cache[1], torch.zeros(0, dtype=torch.int64, device=DEV), "fp8", scales[0], scales[1])
    ops.reshape_and_cache_flash(key, value, cache[0], cache[1], torch.full((3,), -1, device=DEV), "fp8", scales[0], scales[1])
    assert torch.equal(cache.view(torch.uint8), before)


# ---- attention --------------------------------------------------------------------------
LENS = [0, 1, 15, 16, 17, 31, 33, 127, 128, 129, 200, 255, 257, 640, 2]


@pytest.mark.parametrize("dtype", [F32, F, B])
@pytest.mark.parametrize("h,d,bs,pad", [(3, 64, 16, 0), (2, 128, 16, 0), (5, 32, 16, 0), (1, 256, 32, 0), (9, 128, 48, 0), (2, 64, 32, 16), (4, 128, 16, 48)])
def test_decode_against_fp64(h, d, bs, pad, dtype):
    nb, scale = sum(-(-n // bs) for n in LENS) + 3, d ** -0.5
    cache, scales = make_cache(nb, bs, h, d, seed=h, pad=pad)
    tables = make_tables(LENS, bs, nb, seed=d)
    spoil_behind(cache, tables, LENS, bs)
    q = query(len(LENS), h, d, dtype)
    lens = torch.tensor(LENS, dtype=torch.int32, device=DEV)
    got = A.paged_decode_attention(q, cache[0], cache[1], tables, lens, scale, k_scale=scales[0], v_scale=scales[1])
    again = A.paged_decode_attention(q, cache[0], cache[1], tables, lens, scale, k_scale=scales[0], v_scale=scales[1])
    assert torch.equal(got, again)
    ref = attention_reference(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, list(range(len(LENS) + 1)), LENS, scale)
    check(got, ref, dtype)
    A.raise_on_device_status()


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("lens,h,d,bs", [([9000], 3, 128, 16), ([5, 6000], 2, 64, 32), ([700] * 40, 12, 64, 16), ([1] * 300, 2, 128, 16)])
def test_decode_of_long_and_many_requests(lens, h, d, bs, dtype):
    nb = sum(-(-n // bs) for n in lens)
    cache, scales = make_cache(nb, bs, h, d, seed=1)
    tables = make_tables(lens, bs, nb, width=max(-(-n // bs) for n in lens) + 5)
    q = query(len(lens), h, d, dtype, spread=2.0)
    got = A.paged_decode_attention(q, cache[0], cache[1], tables, torch.tensor(lens, dtype=torch.int32, device=DEV), 0.11, k_scale=scales[0], v_scale=scales[1])
    check(got, attention_reference(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, list(range(len(lens) + 1)), lens, 0.11), dtype)


def run_prefix(q, cache, scales, tables, starts, lens, scale, **kw):
    return A.paged_prefix_attention(q, cache[0], cache[1], tables, torch.tensor(starts, dtype=torch.int32, device=DEV),
                                    torch.tensor(lens, dtype=torch.int32, device=DEV), max(b - a for a, b in zip(starts, starts[1:])), scale,
                                    scales[0], scales[1], **kw)


@pytest.mark.parametrize("dtype", [F32, F, B])
@pytest.mark.parametrize("h,d,bs,rows,lens", [
    (2, 128, 16, [1, 16, 17, 5, 0, 130, 64], [1, 16, 40, 300, 20, 130, 257]),
    (3, 64, 16, [129, 3, 1, 200], [700, 3, 129, 201]),
    (2, 64, 32, [2, 3, 4, 5, 6], [33, 64, 65, 900, 6]),
    (1, 256, 16, [20, 7], [50, 7]), (4, 32, 16, [33], [99]),
    (2, 128, 48, [4] * 12, [100 + 7 * i for i in range(12)]),
    (1, 64, 16, [300], [1500]), (2, 128, 16, [9, 4], [5, 0]),
])
def test_prefix_against_fp64(h, d, bs, rows, lens, dtype):
    nb, scale = sum(-(-n // bs) for n in lens) + 1, d ** -0.5
    cache, scales = make_cache(nb, bs, h, d, seed=d)
    tables = make_tables(lens, bs, nb, seed=h)
    spoil_behind(cache, tables, lens, bs)
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    q = query(starts[-1], h, d, dtype)
    got = run_prefix(q, cache, scales, tables, starts, lens, scale)
    assert torch.equal(got, run_prefix(q, cache, scales, tables, starts, lens, scale))
    check(got, attention_reference(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, starts, lens, scale), dtype)
    A.raise_on_device_status()


@pytest.mark.parametrize("d,dtype", [(64, F), (128, B), (32, F32)])
def test_prefix_leaves_rows_of_no_request(d, dtype):
    lens, bs, h = [40, 9], 16, 2
    cache, scales = make_cache(8, bs, h, d)
    tables = make_tables(lens, bs, 8)
    q = query(200, h, d, dtype)
    out = torch.full((200, h * d + 8), 7.0, dtype=dtype, device=DEV)[:, 8:]
    starts = [3, 30, 36]
    assert run_prefix(q, cache, scales, tables, starts, lens, 0.1, out=out) is out
    ref = attention_reference(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, starts, lens, 0.1)
    check(out[3:36], tuple(x[3:36] for x in ref), dtype)
    assert (out[:3] == 7).all() and (out[36:] == 7).all()


@pytest.mark.parametrize("d,dtype,rows", [(64, F, 1), (128, B, 1), (128, F, 20), (64, B, 140), (32, F32, 3)])
def test_pages_outside_the_cache_make_their_rows_nan(d, dtype, rows):
    """Table entries are checked before anything is read through them."""
    lens, bs, h = [300, 300, 300, 20], 16, 2
    nb = 70
    cache, scales = make_cache(nb, bs, h, d)
    tables = make_tables(lens, bs, nb)
    good = tables.clone()
    tables[0, 3], tables[2, 18] = nb, -1
    tables[3, 5] = 2 ** 31 - 1   # behind the last token
    each = [rows, rows, rows, min(rows, 20)]
    starts = [0]
    for n in each:
        starts.append(starts[-1] + n)
    q = query(starts[-1], h, d, dtype)
    got = run_prefix(q, cache, scales, tables, starts, lens, 0.1)
    want = run_prefix(q, cache, scales, good, starts, lens, 0.1)
    assert torch.isnan(got[:rows]).all()
    first = 2 * rows + max(0, rows - 12)    # token 288 and on are in the other one's bad block
    assert torch.isnan(got[first:3 * rows]).all() and torch.equal(got[2 * rows:first], want[2 * rows:first])
    assert torch.equal(got[rows:2 * rows], want[rows:2 * rows]) and torch.equal(got[3 * rows:], want[3 * rows:])
    A.raise_on_device_status()


@pytest.mark.parametrize("d,dtype,rows", [(64, F, 1), (128, B, 9), (128, F, 150), (64, F32, 2)])
def test_values_of_very_different_scales(d, dtype, rows):
    """Blocks whose scales lie 2^60 apart: small values count as what they are where the weight is theirs, zeros stay zeros."""
    lens, bs, h = [200], 16, 2
    cache, scales = make_cache(16, bs, h, d, spread=False)
    tables = make_tables(lens, bs, 16)
    q = query(rows, h, d, dtype)
    ids = tables[0].long()
    scales[1, ids[0]] = 2.0 ** -118
    cache.view(torch.uint8)[1, ids[0]] = 0
    scales[1, ids[1]] *= 2.0 ** -60 if dtype != F else 2.0 ** -10
    scales[1, ids[2]] *= 2.0 ** 12 if dtype != F else 2.0 ** 6
    # nearly all the weight of head 0 on a block of small values
    cache.view(E4M3)[0, ids[1], :, 0] = (q[0, :d].float() / q[0, :d].abs().max() * 400).to(E4M3)
    ref = attention_reference(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, [0, rows], lens, d ** -0.5)
    check(run_prefix(q, cache, scales, tables, [0, rows], lens, d ** -0.5), ref, dtype)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-41])
@pytest.mark.parametrize("rows", [1, 40])
def test_any_scale_of_the_scores(scale, rows):
    lens, bs, h, d = [90, 300], 16, 2, 64
    cache, scales = make_cache(40, bs, h, d)
    tables = make_tables(lens, bs, 40)
    starts = [0, rows, 2 * rows]
    q = query(2 * rows, h, d, F)
    ref = attention_reference(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, starts, lens, scale)
    check(run_prefix(q, cache, scales, tables, starts, lens, scale), ref, F)


@pytest.mark.parametrize("d,dtype,rows", [(64, F, 1), (128, B, 3), (128, F, 150)])
def test_growing_scores(d, dtype, rows):
    """Scores that grow by far more than 2^8 along the tokens."""
    lens, bs, h = [700], 16, 2
    cache, scales = make_cache(44, bs, h, d, spread=False)
    tables = make_tables(lens, bs, 44)
    scales[0, tables[0].long()] *= torch.linspace(0.0, 6.0, 44, device=DEV)[:, None]
    q = query(rows, h, d, dtype, spread=3.0)
    ref = attention_reference(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, [0, rows], lens, 0.3)
    check(run_prefix(q, cache, scales, tables, [0, rows], lens, 0.3), ref, dtype)


def test_nan_in_a_query_and_in_the_cache():
    lens, bs, h, d = [200, 150], 16, 2, 64
    for rows, dtype in ((1, F), (30, B), (140, F)):
        cache, scales = make_cache(40, bs, h, d)
        tables = make_tables(lens, bs, 40)
        starts = [0, rows, 2 * rows]
        q = query(2 * rows, h, d, dtype).contiguous()
        want = run_prefix(q, cache, scales, tables, starts, lens, 0.1)
        q[0, 3] = float("nan")
        got = run_prefix(q, cache, scales, tables, starts, lens, 0.1)
        assert torch.isnan(got[0, :d]).all() and torch.equal(got[0, d:], want[0, d:]) and torch.equal(got[1:], want[1:])
        q[0, 3] = 0.5
        cache.view(torch.uint8)[1, tables[1, 0].long(), 2, 1, 5] = 0x7f   # a value row that every row of the second request sees
        got = run_prefix(q, cache, scales, tables, starts, lens, 0.1)
        assert torch.isnan(got[rows:, d + 5]).all() and not torch.isnan(got[:rows]).any()
        assert torch.equal(got[rows:, :d], want[rows:, :d])


# ---- together ---------------------------------------------------------------------------
def test_captured_calls_replay_on_another_stream():
    lens, bs, h, d = [37, 300, 16], 16, 2, 128
    cache, scales = make_cache(40, bs, h, d)
    tables, seq = make_tables(lens, bs, 40), torch.tensor(lens, dtype=torch.int32, device=DEV)
    key, value = rows_of(3, h, d, F, seed=2)
    slots = torch.stack([tables[r, (n - 1) // bs].long() * bs + (n - 1) % bs for r, n in enumerate(lens)])
    q = query(3, h, d, F).contiguous()
    ws = torch.empty(8 << 20, dtype=torch.uint8, device=DEV)

    def step(c, s):
        ops.reshape_and_cache_flash(key, value, c[0], c[1], slots, "fp8", s[0], s[1])
        return A.paged_decode_attention(q, c[0], c[1], tables, seq, 0.1, workspace=ws, k_scale=s[0], v_scale=s[1])
    want_c, want_s = cache.clone(), scales.clone()
    step(cache.clone(), scales.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache, scales)
    for seed in (5, 6):
        k2, v2 = rows_of(3, h, d, F, seed=seed)
        key.copy_(k2), value.copy_(v2)
        q.copy_(query(3, h, d, F, seed=seed))
        want = step(want_c, want_s).clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        assert torch.equal(out, want) and same_codes(cache, want_c) and torch.equal(scales, want_s)


def test_prompts_are_written_beside_attention_on_another_stream_and_captured():
    """A write of many rows has scratch of its own: attention on another stream is not disturbed, nor is a replay by a later call."""
    lens, bs, h, d = [3000, 700], 16, 2, 128
    cache, scales = make_cache(240, bs, h, d)
    tables, seq, q = make_tables(lens, bs, 240), torch.tensor(lens, dtype=torch.int32, device=DEV), query(2, h, d, F)
    key, value = rows_of(1500, h, d, F, seed=2)
    slots = torch.arange(1500, device=DEV)

    def write(c, s):
        ops.reshape_and_cache_flash(key, value, c[0], c[1], slots, "fp8", s[0], s[1])

    def attend():
        return A.paged_decode_attention(q, cache[0], cache[1], tables, seq, 0.1, k_scale=scales[0], v_scale=scales[1])
    before = [make_cache(100, bs, h, d, seed=3) for _ in range(3)]
    want_c, want_s = before[0]
    write(want_c, want_s)
    want, side = attend(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(8):
        with torch.cuda.stream(side):
            write(*before[1])
        outs.append(attend())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs) and same_codes(before[1][0], want_c) and torch.equal(before[1][1], want_s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        write(*before[2])
    key.copy_(rows_of(1500, h, d, F, seed=4)[0])
    write(want_c, want_s)
    graph.replay()
    torch.cuda.synchronize()
    assert same_codes(before[2][0], want_c) and torch.equal(before[2][1], want_s)


@pytest.mark.parametrize("rows", [[3, 1], [30, 200]])
def test_the_bound_of_a_requests_rows_may_be_far_too_large(rows):
    lens, bs, h, d = [100, 900], 16, 2, 64
    cache, scales = make_cache(80, bs, h, d)
    tables, seq = make_tables(lens, bs, 80), torch.tensor(lens, dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, rows[0], sum(rows)], dtype=torch.int32, device=DEV)
    q = query(sum(rows), h, d, F)
    ref = attention_reference(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, starts.tolist(), lens, 0.1)
    for most in (max(rows), 2 ** 20, 2 ** 31 - 1):
        check(A.paged_prefix_attention(q, cache[0], cache[1], tables, starts, seq, most, 0.1, scales[0], scales[1]), ref, F)


class _Fp8:
    cache_dtype, sliding_window = "fp8", None


def metadata(rows, lens, tables, slots, prefix):
    """Prompt rows (`rows` of each request, some behind a cached prefix) or, rows == None, one decode token of each."""
    none, dev = slots[:0], dict(dtype=torch.int32, device=DEV)
    n = len(lens)
    base = dict(num_hidden_cache_tokens=0, num_tot_tokens=slots.numel(), slot_mapping=slots, slot_mapping_shared=none, hidden_cache_use_tot=none,
                kv_cache_use_tot=none, hidden_cache_use_input=none, hidden_cache_store_tot=none, hidden_holder_upd=none, hidden_holder_pull=none,
                seq_lens=list(lens), seq_lens_tensor=torch.tensor(lens, **dev), use_cuda_graph=False)
    if rows is None:
        return A.FlashAttentionMetadata(num_prefills=0, num_prefill_tokens=0, num_decode_tokens=n, max_query_len=1, max_prefill_seq_len=0,
                                        max_decode_seq_len=max(lens), query_start_loc=None, seq_start_loc=None, context_lens_tensor=None,
                                        block_tables=tables, **base)
    starts = torch.tensor([0] + rows, **dev).cumsum(0).to(torch.int32)
    return A.FlashAttentionMetadata(num_prefills=n, num_prefill_tokens=sum(rows), num_decode_tokens=0, max_query_len=max(rows),
                                    max_prefill_seq_len=max(lens), max_decode_seq_len=0, query_start_loc=starts,
                                    seq_start_loc=torch.tensor([0] + list(lens), **dev).cumsum(0).to(torch.int32),
                                    context_lens_tensor=torch.tensor([a - b for a, b in zip(lens, rows)], **dev),
                                    block_tables=tables if prefix else torch.zeros(n, 0, **dev), **base)


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("h,d", [(4, 64), (2, 128)])
def test_a_layer_serves_requests_from_an_8_bit_cache(h, d, dtype):
    """Prompts, a second turn behind them, decode steps, a block copy and a swap out and in, through the layer and the cache engine:
    every attention output against 64 bits over the cache as the definition has it."""
    e, bs, nb = h * d, 16, 32
    g = torch.Generator(device=DEV).manual_seed(h)
    w = torch.randn(3 * e, e, generator=g, device=DEV).mul_(e ** -0.5).to(dtype)
    eye = torch.eye(e, device=DEV, dtype=dtype)
    layer = OPTAttention(e, h, w, None, eye, None, cache_config=_Fp8)
    engine = CacheEngine(1, h, d, bs, nb, 4, E4M3, device=DEV)
    cache, scales = engine.gpu_cache[0], engine.gpu_scale[0]
    want = [(cache[p].cpu().view(torch.uint8).clone(), scales[p].cpu().clone()) for p in (0, 1)]
    lens, total = [0, 0, 0], [70, 90, 45]
    tables = make_tables(total, bs, nb)
    first = [37, 16, 1]

    def advance(rows, prefix):
        pos = [(r, p) for r, n in enumerate(rows) for p in range(lens[r], lens[r] + n)]
        slots = torch.tensor([int(tables[r, p // bs]) * bs + p % bs for r, p in pos], device=DEV, dtype=torch.int64)
        for r, n in enumerate(rows):
            lens[r] += n
        x = torch.randn(len(pos), e, generator=g, device=DEV).to(dtype)
        meta = metadata(rows if prefix is not None else None, lens, tables, slots, prefix)
        got = layer(x, cache, None, meta, kv_scale=scales)
        q, k, v = layer.qkv_proj(x)[0].chunk(3, dim=1)
        for p, y in ((0, k), (1, v)):
            write_reference(*want[p], y.reshape(-1, h, d).cpu(), slots.tolist(), bs)
            assert same_codes(cache[p], want[p][0]) and torch.equal(scales[p].cpu(), want[p][1])
        if prefix is False:
            return   # prompts attend to their rows as they are: the test of that attention is elsewhere
        starts = [0]
        for n in rows:
            starts.append(starts[-1] + n)
        ref = attention_reference(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, starts, lens, d ** -0.5)
        check(got, ref, dtype)   # o_proj is the identity
    advance(first, False)
    advance([20, 33, 18], True)
    for _ in range(9):
        advance([1, 1, 1], None)
    src, dst = int(tables[0, 0]), [b for b in range(nb) if b not in tables[:, :6].flatten().tolist()][0]
    engine.copy(torch.tensor([[src, dst]], device=DEV))
    tables[0, 0] = dst
    for p in (0, 1):
        want[p][0][dst], want[p][1][dst] = want[p][0][src].clone(), want[p][1][src].clone()
    advance([1, 1, 1], None)
    engine.swap_out(torch.tensor([[int(tables[1, 0]), 2]]))
    cache.view(torch.uint8)[:, int(tables[1, 0])] = 0x55
    scales[:, int(tables[1, 0])] = 3.0
    engine.swap_in(torch.tensor([[2, int(tables[1, 0])]]))
    advance([1, 1, 1], None)
    A.raise_on_device_status()


def test_padded_decode_batches_and_mixed_ones():
    """A decode batch padded for a graph (slot -1, length 0) and a batch of prompt chunks and decode tokens, through the backend."""
    h, d, bs, nb = 3, 64, 16, 40
    cache, scales = make_cache(nb, bs, h, d, seed=8)
    impl = A.FlashAttentionImpl(h, d, 0.125, h, None, None, "fp8_e4m3")
    lens = [40, 17, 0, 0]
    tables = make_tables([40, 17, 0, 0], bs, nb)
    slots = torch.tensor([int(tables[0, 2]) * bs + 7, int(tables[1, 1]) * bs, -1, -1], device=DEV)
    q, (k, v) = query(4, h, d, F), rows_of(4, h, d, F, seed=3)
    want = [(cache[p].cpu().view(torch.uint8).clone(), scales[p].cpu().clone()) for p in (0, 1)]
    for p, rows in ((0, k), (1, v)):
        write_reference(*want[p], rows.cpu(), slots.tolist(), bs)
    meta = metadata(None, lens, tables, slots, None)
    got = impl.forward(q, k.reshape(4, -1), v.reshape(4, -1), cache, None, meta, scales)
    for p in (0, 1):
        assert same_codes(cache[p], want[p][0]) and torch.equal(scales[p].cpu(), want[p][1])
    check(got, attention_reference(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, list(range(5)), lens, 0.125), F)
    assert (got[2:] == 0).all()

    rows, lens = [30, 5, 1, 1], [50, 5, 33, 17]   # two chunks of prompts, two decode tokens
    tables = make_tables(lens, bs, nb, seed=4)
    pos = [(r, p) for r, n in enumerate(rows) for p in range(lens[r] - n, lens[r])]
    slots = torch.tensor([int(tables[r, p // bs]) * bs + p % bs for r, p in pos], device=DEV)
    t = len(pos)
    q, (k, v) = query(t, h, d, B), rows_of(t, h, d, B, seed=5)
    pre = metadata(rows[:2], lens[:2], tables[:2], slots, True)
    meta = A.replace(pre, num_prefills=2, num_prefill_tokens=35, num_decode_tokens=2, num_tot_tokens=t, seq_lens=lens,
                     seq_lens_tensor=torch.tensor(lens, dtype=torch.int32, device=DEV), block_tables=tables, max_decode_seq_len=33,
                     context_lens_tensor=torch.tensor([20, 0, 32, 16], dtype=torch.int32, device=DEV))
    got = impl.forward(q, k.reshape(t, -1), v.reshape(t, -1), cache, None, meta, scales)
    ref = attention_reference(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, [0, 30, 35, 36, 37], lens, 0.125)
    check(got, ref, B)


def test_what_the_backend_refuses():
    h, d, bs = 2, 64, 16
    cache, scales = make_cache(8, bs, h, d)
    impl = A.FlashAttentionImpl(h, d, 0.125, h, None, None, "fp8")
    tables = make_tables([20], bs, 8)
    slots = torch.tensor([int(tables[0, 1]) * bs + 3], device=DEV)
    q, (k, v) = query(1, h, d, F), rows_of(1, h, d, F, seed=1)
    meta = metadata(None, [20], tables, slots, None)
    with pytest.raises(ValueError, match="kv_scale"):
        impl.forward(q, k.reshape(1, -1), v.reshape(1, -1), cache, None, meta)
    with pytest.raises(RuntimeError, match="float32"):
        impl.forward(q, k.reshape(1, -1), v.reshape(1, -1), cache, None, meta, scales.double())
    with pytest.raises(ValueError, match="float8_e4m3fn or uint8"):
        impl.forward(q, k.reshape(1, -1), v.reshape(1, -1), cache.view(E4M3).half(), None, meta, scales)
    with pytest.raises(AssertionError, match="kv_scale"):
        A.FlashAttentionImpl(h, d, 0.125, h, None, None, "auto").forward(q, k.reshape(1, -1), v.reshape(1, -1), cache.half(), None, meta, scales)


@pytest.mark.parametrize("rows,dtype", [(1, F), (1, F32), (7, B), (12, F), (40, B), (200, F)])
def test_rows_of_unaligned_tensors(rows, dtype):
    """Query and output rows that no vector load takes."""
    lens, bs, h, d = [260, 300], 16, 3, 64
    cache, scales = make_cache(40, bs, h, d)
    tables = make_tables(lens, bs, 40)
    starts = [0, rows, 2 * rows]
    wide = torch.randn(2 * rows, h * d + 5, device=DEV).to(dtype)
    q, out = wide[:, 3:3 + h * d], torch.zeros(2 * rows, h * d + 3, dtype=dtype, device=DEV)[:, 1:1 + h * d]
    run_prefix(q, cache, scales, tables, starts, lens, 0.1, out=out)
    check(out, attention_reference(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, starts, lens, 0.1), dtype)


# ---- many rows --------------------------------------------------------------------------
def attention_reference_by_request(q, k8, v8, ks, vs, tables, starts, lens, scale):
    """`attention_reference` with all of a request's rows at a time."""
    t, h, d = q.shape
    bs, most = k8.shape[1], tables.shape[1] * k8.shape[1]
    out, size, least = (torch.full((t, h, d), float("nan"), dtype=torch.double, device=DEV) for _ in range(3))
    score, count = torch.zeros(t, h, 1, dtype=torch.double, device=DEV), torch.zeros(t, 1, 1, dtype=torch.double, device=DEV)
    for r, n in enumerate(lens):
        a, b = starts[r], starts[r + 1]
        n = max(0, min(n, most))
        if n == 0:
            out[a:b] = size[a:b] = least[a:b] = 0.0
        if a == b or n == 0:
            continue
        ids = tables[r, :-(-n // bs)].long()
        k, v = ((c.view(torch.uint8)[ids].view(E4M3).double() * s[ids].double()[:, None, :, None]).flatten(0, 1)[:n].transpose(0, 1)
                for c, s in ((k8, ks), (v8, vs)))                                                             # [H, n, D]
        codes = v8.view(torch.uint8)[ids].view(E4M3).double().abs().flatten(0, 1)[:n].transpose(0, 1)
        steps = vs[ids].double().repeat_interleave(bs, 0)[:n].transpose(0, 1)
        x = q[a:b].double().transpose(0, 1)                                                                   # [H, rows, D]
        keys = n - (b - 1 - torch.arange(a, b, device=DEV))
        seen = torch.arange(n, device=DEV)[None, :] < keys[:, None]
        p = torch.softmax((x @ k.transpose(1, 2) * scale).masked_fill(~seen, -float("inf")), dim=2).nan_to_num(0.0)
        out[a:b], size[a:b] = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
        least[a:b] = (2.0 ** -32 * (p * steps[:, None]).amax(2, keepdim=True) * (seen.double() @ codes)).transpose(0, 1)
        score[a:b, :, 0] = ((x.abs() @ k.abs().transpose(1, 2) * abs(scale)) * seen).amax(2).transpose(0, 1)
        count[a:b, 0, 0] = keys.clamp_min(0).double()
    return out, size, score, count, least


def check_prefix(h, d, rows, lens, dtype, bs=16, scale=None):
    nb, scale = sum(-(-n // bs) for n in lens) + 1, d ** -0.5 if scale is None else scale
    cache, scales = make_cache(nb, bs, h, d, seed=d)
    tables = make_tables(lens, bs, nb, seed=h)
    spoil_behind(cache, tables, lens, bs)
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    q = query(starts[-1], h, d, dtype)
    got = run_prefix(q, cache, scales, tables, starts, lens, scale)
    for _ in range(3):
        assert torch.equal(got, run_prefix(q, cache, scales, tables, starts, lens, scale))
    check(got, attention_reference_by_request(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, starts, lens, scale), dtype)
    A.raise_on_device_status()


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("h,d", [(2, 64), (20, 64), (2, 128), (20, 128)])
@pytest.mark.parametrize("rows,lens", [([520, 500], [700, 900]), ([257, 255, 200], [300, 256, 1100])])
def test_pairs_of_row_tiles_of_which_the_second_is_empty(rows, lens, h, d, dtype):
    """Two row tiles share a CTA; a request's last 1 ... 128 rows fill the first one alone.  Two heads: the tokens are cut into parts, too."""
    check_prefix(h, d, rows, lens, dtype)


@pytest.mark.parametrize("tokens", [1000, 2048, 6000])
@pytest.mark.parametrize("d,dtype,rows", [(64, F, 1), (128, B, 5), (64, B, 12), (128, F, 20), (64, F32, 2)])
def test_a_whole_part_outside_the_cache_makes_its_rows_nan(d, dtype, rows, tokens):
    """Tokens 512 ... 1023 are a part of their own, or several, in every kernel; two to eight parts, and more, are joined."""
    bs, h, nb = 16, 2, -(-tokens // 16)
    cache, scales = make_cache(nb, bs, h, d)
    tables = make_tables([tokens], bs, nb)
    q = query(rows, h, d, dtype)
    want = run_prefix(q, cache, scales, tables, [0, rows], [tokens], 0.1)
    assert not torch.isnan(want).any()
    bad = tables.clone()
    bad[0, 32:64] = nb
    assert torch.isnan(run_prefix(q, cache, scales, bad, [0, rows], [tokens], 0.1)).all()
    scales[0, tables[0, 32:64].long(), 0] = float("nan")
    got = run_prefix(q, cache, scales, tables, [0, rows], [tokens], 0.1)
    assert torch.isnan(got[:, :d]).all() and torch.equal(got[:, d:], want[:, d:])
    A.raise_on_device_status()


@pytest.mark.parametrize("width", [None, 400])   # the latter's tokens are cut into more than eight parts
@pytest.mark.parametrize("most", [0, 1, 5, 12, 20, 130, 300])
@pytest.mark.parametrize("d,dtype", [(64, F), (128, B), (64, F32)])
def test_rows_beyond_the_bound_of_a_requests_rows_are_left(d, dtype, most, width):
    lens, rows, bs, h = [400, 350, 9], [310, 4, 9], 16, 2
    cache, scales = make_cache(60, bs, h, d)
    tables, seq = make_tables(lens, bs, 60, width=width), torch.tensor(lens, dtype=torch.int32, device=DEV)
    starts = [0, 310, 314, 323]
    q = query(323, h, d, dtype)
    out = torch.full((323, h * d), 7.0, dtype=dtype, device=DEV)
    A.paged_prefix_attention(q, cache[0], cache[1], tables, torch.tensor(starts, dtype=torch.int32, device=DEV), seq, most, 0.1, scales[0], scales[1],
                             out=out)
    within = torch.cat([torch.arange(n) < most for n in rows]).to(DEV)
    assert (out[~within] == 7).all()
    ref = attention_reference_by_request(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, starts, lens, 0.1)
    check(out[within], tuple(x[within] for x in ref), dtype)
    A.raise_on_device_status()


@pytest.mark.parametrize("d,dtype,rows", [(64, B, 1), (128, B, 7), (128, B, 12), (64, B, 60), (128, B, 200), (64, F32, 3)])
def test_values_of_the_least_scale(d, dtype, rows):
    """Outputs near 2^-112 are bf16 numbers like any other."""
    lens, bs, h = [900], 16, 3
    cache, scales = make_cache(60, bs, h, d)
    tables = make_tables(lens, bs, 60)
    scales[1] = 2.0 ** -118
    q = query(rows, h, d, dtype)
    ref = attention_reference_by_request(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, [0, rows], lens, 0.1)
    check(run_prefix(q, cache, scales, tables, [0, rows], lens, 0.1), ref, dtype)


def test_a_captured_call_keeps_its_scratch_when_a_later_one_needs_more(monkeypatch):
    monkeypatch.setattr(A, "_workspaces", {})
    lens, bs, h, d = [9000], 16, 4, 128
    cache, scales = make_cache(563, bs, h, d)
    tables, seq, q = make_tables(lens, bs, 563), torch.tensor(lens, dtype=torch.int32, device=DEV), query(1, h, d, F)

    def attend(n=1):
        return A.paged_decode_attention(q.repeat(n, 1), cache[0], cache[1], tables.repeat(n, 1), seq.repeat(n), 0.1,
                                        k_scale=scales[0], v_scale=scales[1])
    want = attend()
    size = A._workspaces[q.device].numel()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend()
    attend(64)
    assert A._workspaces[q.device].numel() > size
    torch.cuda.synchronize()
    others = [torch.zeros(size, dtype=torch.uint8, device=DEV) for _ in range(4)]   # what the allocator has free of that size
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and not any(x.any() for x in others)


_STATUS = """
import torch
from torch.profiler import ProfilerActivity, profile
from apt_serve_b200 import attention as A, ops
dev = torch.device("cuda", 0)

def copies():
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        A.cache_ops_status(dev)
    return sum(e.name.startswith("Memcpy DtoH") for e in p.events())
x, slots = torch.zeros(2, 2, 64, device=dev, dtype=torch.float16), torch.tensor([3, 99], device=dev)
A.cache_ops_status(dev)
before = copies()
cache, scales = torch.zeros(2, 4, 16, 2, 64, device=dev, dtype=torch.float8_e4m3fn), torch.zeros(2, 4, 2, device=dev)
ops.reshape_and_cache_flash(x, x, cache[0], cache[1], slots, "fp8", scales[0], scales[1])
assert A.cache_ops_status(dev) == 2 and A.cache_ops_status(dev) == 0
print("copies", before, copies())
"""


def test_reading_the_status_costs_no_more_where_no_8_bit_cache_is_written():
    """Every word of the status is a copy to the host that is waited for."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _STATUS], cwd=root, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
    if "copies 0 0" in r.stdout:
        pytest.skip("no activity records on this machine")
    assert "copies 3 4" in r.stdout, r.stdout


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("h,d,rows,lens", [
    (2, 64, [1000], [3000]), (20, 128, [700, 690, 650], [700, 2000, 651]),   # several pairs of row tiles a request
    (1, 64, [129 + r % 7 for r in range(260)], [140 + r % 50 for r in range(260)]),   # more pairs than are put in order
    (1, 128, [17 + r % 3 for r in range(300)], [30 + r % 90 for r in range(300)]),    # as many single tiles
])
def test_prefix_of_many_rows_and_requests(h, d, rows, lens, dtype):
    check_prefix(h, d, rows, lens, dtype)


@pytest.mark.parametrize("dtype", [F32, F, B])
@pytest.mark.parametrize("h,d,bs", [(3, 64, 16), (2, 128, 32), (1, 256, 16), (5, 32, 16)])
def test_a_decode_step_in_one_call(h, d, bs, dtype):
    """Ragged requests, one that begins a block, one of a single token, one longer than a part; several steps."""
    lens, nb = [40, 33, 1, 700, 16], 60
    cache, scales = make_cache(nb, bs, h, d, seed=6)
    impl = A.FlashAttentionImpl(h, d, 0.11, h, None, None, "fp8")
    tables = make_tables([n + 3 for n in lens], bs, nb)
    for step in range(3):
        now = [n + step for n in lens]
        slots = torch.tensor([int(tables[r, (n - 1) // bs]) * bs + (n - 1) % bs for r, n in enumerate(now)], device=DEV)
        q, (k, v) = query(5, h, d, dtype, seed=step), rows_of(5, h, d, dtype, seed=step)
        want = [(cache[p].cpu().view(torch.uint8).clone(), scales[p].cpu().clone()) for p in (0, 1)]
        for p, rows in ((0, k), (1, v)):
            write_reference(*want[p], rows.cpu(), slots.tolist(), bs)
        meta = metadata(None, now, tables, slots, None)
        got = impl._plain_decode_fp8(q, k.reshape(5, -1), v.reshape(5, -1), cache, meta, scales)
        assert got is not None
        for p in (0, 1):
            assert same_codes(cache[p], want[p][0]) and torch.equal(scales[p].cpu(), want[p][1])
        check(got, attention_reference(q.reshape(-1, h, d), cache[0], cache[1], scales[0], scales[1], tables, list(range(6)), now, 0.11), dtype)
    A.raise_on_device_status()
