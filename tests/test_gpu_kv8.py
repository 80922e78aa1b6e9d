"""The paged 8-bit K/V cache on the GPU: write, read, attention over all tokens and
over listed chunks, against the 64-bit restatement in oracle/kv8.py.

Bytes and scales are compared for equality: with power-of-two scales the written
byte is one rounding of an exact quotient.  Attention is held to a bound per
value, out of what is rounded on the way to it (see ``bound``)."""
import threading

import numpy as np
import pytest
import torch

from csahca_amd import extension, kv8_layout, native
from oracle import kv8 as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("no HIP device visible")
    native.lib()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def filled(pages, H, page, D, fmt, seed, spread=3):
    """A cache of random bytes (no NaN) and scales 2^-spread..2^spread."""
    g = gen(seed)
    code = torch.randint(0, 256, (2, pages * H * page * D), generator=g, dtype=torch.uint8)
    if fmt == E4M3:
        code[(code & 127) == 127] -= 1
    else:
        code[code == 128] = 129
    k = code[0].view(fmt).view(pages, H, page, D)
    v = code[1].view(fmt).view(pages, H, page // 16, D, 16)
    down = -8 if fmt == E4M3 else -6
    ks, vs = (torch.pow(2.0, torch.randint(down - spread, down + spread + 1, (pages, H), generator=g).float())
              for _ in range(2))
    return kv8_layout.Kv8Cache(k, v, ks, vs)


def to_gpu(cache):
    return tuple(t.to(DEV) for t in cache)


def table_of(B, blocks, pages, seed):
    return torch.randperm(pages, generator=gen(seed))[: B * blocks].view(B, blocks).to(torch.int32)


def same_bytes(got, want):
    for name, a, b in zip(kv8_layout.Kv8Cache._fields, got, want):
        x, y = a.cpu().view(torch.uint8).numpy().ravel(), b.view(torch.uint8).numpy().ravel()
        bad = np.flatnonzero(x != y)
        assert bad.size == 0, f"{name}: {bad.size} of {x.size} bytes differ, first at {bad[:4]}: {x[bad[:4]]} {y[bad[:4]]}"


def bound(want, mass, size, dtype, D, n, peak):
    """Error of one output value, from the roundings on the way to it:

    * the result: half a step of its type, which below the least normal value is
      half the least subnormal (f16: 2^-25);
    * every weight p: beside 16-bit values one rounding to f16's 11 bits, and where
      f16 has no exponent for it half its least step: weights are held times 2^12
      beside the largest, the step is 2^-24, so 2^-36 of the largest weight a token,
      n 2^-36 ``peak`` in all; beside f32 24 bits and nothing lost.  "Largest" is
      by p times its page's V scale; where those differ by up to 2^10 the sum's
      weights are the same ones, so it may miss n 2^-26 of itself;
    * p's own relative error, twice (numerator, sum): the score's |q| |k| products
      in fp32 (D + 8 roundings), 4 roundings of a score of that size and the
      exponential's two;
    * sums over n tokens in fp32, in pieces of at most 64 terms at a time and
      their rescalings."""
    half, least = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    p_bits = 2.0 ** -23 if dtype == F32 else 2.0 ** -11
    lost = 0.0 if dtype == F32 else n * (peak * 2.0 ** -36 + np.abs(want) * 2.0 ** -26)
    score = size[..., None] * (D + 12) * 2.0 ** -24 + 2.0 ** -21
    sums = (64 + n / 16) * 2.0 ** -24
    return half * np.abs(want) + mass * (p_bits + 2 * score + 2 * sums) + lost + least


def peak_of(cache):
    return plain.LARGEST[cache[0].dtype] * float(cache[3].max())


def close(got, want, mass, size, n, peak):
    """``peak``: the largest |v| that the scales allow."""
    g = got.double().cpu().numpy()
    tol = bound(want, mass, size, got.dtype, got.shape[-1], n, peak)
    # beyond the type's largest value (f16: from 65520 on) the rounded result is an infinity
    over = np.isinf(torch.from_numpy(want).to(got.dtype).double().numpy())
    bad = np.where(over, g != np.copysign(np.inf, want), ~(np.abs(g - want) <= tol))
    if bad.any():
        pytest.fail(f"{bad.sum()} of {bad.size} values off, worst {np.nanmax(np.abs(g - want) / tol):.3g} of the "
                    f"bound, first at {np.argwhere(bad)[0]}: {g[bad][:3]} {want[bad][:3]}")


# ---------------------------------------------------------------------------
# write
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,page,N,start", [
    (32, 16, 1, (0, 5, 15)), (64, 16, 1, (16, 31, 33)), (96, 48, 50, (0, 47, 95)), (128, 64, 1, (63, 64, 127)),
    (128, 64, 130, (0, 1, 63)), (160, 32, 33, (31, 32, 0)), (192, 256, 300, (250, 3, 16)), (256, 128, 7, (125, 126, 0)),
    (224, 64, 65, (60, 64, 0)), (128, 16, 40, (8, 15, 2)),
])
def test_write(fmt, dtype, D, page, N, start):
    B, H = 3, 2
    blocks = (max(start) + N) // page + 1
    pages = B * blocks + 2
    cache = filled(pages, H, page, D, fmt, seed=N)
    table = table_of(B, blocks, pages, seed=page)
    g = gen(D + N)
    k, v = (torch.randn(B, H, N, D, generator=g) * torch.pow(2.0, torch.randint(-6, 7, (B, H, 1, 1), generator=g).float())
            for _ in range(2))
    k, v = k.to(dtype), v.to(dtype)
    start = torch.tensor(start, dtype=torch.int32)
    want = plain.write(k, v, cache, table, start)
    got = to_gpu(cache)
    native.kv8_write(k.to(DEV), v.to(DEV), *got, table.to(DEV), start.to(DEV))
    same_bytes(got, want)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
def test_write_ragged_strided_and_skipped(fmt):
    """Counts of 0, some, all and out of range; K and V as slices of one
    projection; a negative start, a page outside the pool, positions past the table."""
    B, H, N, D, page, blocks = 7, 3, 37, 64, 16, 4
    pages = B * blocks
    cache = filled(pages, H, page, D, fmt, seed=5)
    table = table_of(B, blocks, pages, seed=6)
    table[4, 1], table[4, 2] = -1, pages
    start = torch.tensor([0, 17, 30, -3, 3, 60, 11], dtype=torch.int32)
    counts = torch.tensor([0, 5, 37, 20, 37, 37, 99], dtype=torch.int32)
    x = torch.randn(B, N, 3, H, D, generator=gen(8)).to(BF16)
    k, v = x[:, :, 1].transpose(1, 2), x[:, :, 2].transpose(1, 2)
    want = plain.write(k, v, cache, table, start, counts)
    got = to_gpu(cache)
    xg = x.to(DEV)
    native.kv8_write(xg[:, :, 1].transpose(1, 2), xg[:, :, 2].transpose(1, 2), *got, table.to(DEV), start.to(DEV),
                     counts=counts.to(DEV))
    same_bytes(got, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_write_rows_that_no_wide_load_is_aligned_for(dtype, offset):
    B, H, N, D, page = 2, 2, 21, 96, 32
    cache = filled(4, H, page, D, E4M3, seed=1)
    table = table_of(B, 2, 4, seed=2)
    start = torch.tensor([9, 0], dtype=torch.int32)
    flat = torch.randn(2, B * N * H * (D + offset) + offset, generator=gen(offset)).to(dtype)
    k, v = (f[offset:].view(B, N, H, D + offset)[..., :D].transpose(1, 2) for f in flat)
    want = plain.write(k, v, cache, table, start)
    got = to_gpu(cache)
    kg, vg = (f[offset:].view(B, N, H, D + offset)[..., :D].transpose(1, 2) for f in flat.to(DEV))
    native.kv8_write(kg, vg, *got, table.to(DEV), start.to(DEV))
    same_bytes(got, want)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_write_special_values(fmt, dtype):
    """NaN and infinities beside finite values, alone on a page, all zeros,
    subnormals, the largest values, maxima on and beside a power-of-two border,
    values on rounding ties."""
    H, N, D, page = 1, 160, 32, 16
    x = torch.randn(1, H, N, D, generator=gen(3))
    top = plain.LARGEST[fmt]
    x[0, 0, 0, :3] = torch.tensor([float("nan"), float("inf"), -float("inf")])
    x[0, 0, 16:32] = float("nan")
    x[0, 0, 32:48] = float("inf")
    x[0, 0, 48:64] = 0.0
    x[0, 0, 64:80] = torch.finfo(dtype).tiny * torch.rand(16, D, generator=gen(4))
    x[0, 0, 80:96] = torch.finfo(dtype).max
    x[0, 0, 96:112] = top / 64
    x[0, 0, 112:128] = top / 64 * (1 + torch.finfo(dtype).eps)
    x[0, 0, 128:144] = torch.arange(16 * D).view(16, D) / 16
    x[0, 0, 144:160] = -torch.arange(16 * D).view(16, D) * 2.0 ** -11
    x = x.to(dtype)
    cache = filled(N // page, H, page, D, fmt, seed=4)
    table = table_of(1, N // page, N // page, seed=7)
    start = torch.zeros(1, dtype=torch.int32)
    want = plain.write(x, -x, cache, table, start)
    got = to_gpu(cache)
    native.kv8_write(x.to(DEV), -x.to(DEV), *got, table.to(DEV), start.to(DEV))
    if fmt == E4M3:  # a NaN's sign is not part of the format's contract
        got = tuple(t.cpu() for t in got)
        for a, b in ((got[0], want[0]), (got[1], want[1])):
            a, b = a.view(torch.uint8), b.view(torch.uint8)
            nan = (b & 127) == 127
            assert torch.equal(nan, (a & 127) == 127)
            a[nan] = b[nan]
    same_bytes(got, want)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
def test_write_token_by_token_is_the_restated_sequence(fmt):
    """A page filled one token at a time, magnitudes rising and falling: each
    rise rounds what is there anew."""
    B, H, D, page = 2, 2, 32, 16
    cache = filled(4, H, page, D, fmt, seed=9)
    table = table_of(B, 2, 4, seed=10)
    got, want = to_gpu(cache), cache
    g = gen(11)
    for t in range(20):
        mag = 2.0 ** ((t * 7) % 11 - 5)
        k, v = (torch.randn(B, H, 1, D, generator=g).mul(mag).to(BF16) for _ in range(2))
        start = torch.tensor([t, t + 3], dtype=torch.int32)
        want = plain.write(k, v, want, table, start)
        native.kv8_write(k.to(DEV), v.to(DEV), *got, table.to(DEV), start.to(DEV))
        same_bytes(got, want)


def test_write_nothing():
    cache = to_gpu(filled(2, 2, 16, 32, E4M3, seed=1))
    before = [t.clone() for t in cache]
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    for B, N in ((1, 0), (0, 4)):
        x = torch.zeros(B, 2, N, 32, dtype=BF16, device=DEV)
        native.kv8_write(x, x, *cache, table[:B], one[:B])
    x = torch.ones(1, 2, 4, 32, dtype=BF16, device=DEV)
    native.kv8_write(x, x, *cache, table[:, :0], one)
    for a, b in zip(cache, before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ---------------------------------------------------------------------------
# read
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,page,N,start", [(32, 16, 1, None), (64, 48, 50, (0, 7, 95)), (128, 64, 130, (64, 1, -5)),
                                            (256, 256, 70, (250, 16, 0)), (96, 16, 37, (3, 200, 8)),
                                            (224, 32, 65, None)])
def test_read(fmt, dtype, D, page, N, start):
    B, H = 3, 2
    blocks = -(-120 // page)
    pages = B * blocks + 1
    cache = filled(pages, H, page, D, fmt, seed=D)
    table = table_of(B, blocks, pages, seed=N)
    if blocks > 2:
        table[1, 1], table[2, 2] = -1, pages
    lengths = torch.tensor([113, 0, 5 if N == 1 else 2000], dtype=torch.int32)
    start = None if start is None else torch.tensor(start, dtype=torch.int32)
    k, v = native.kv8_read(*to_gpu(cache), table.to(DEV), lengths.to(DEV), N, dtype=dtype,
                           start=None if start is None else start.to(DEV))
    wk, wv = plain.read(cache, table, lengths, N, start)
    for got, want in ((k, wk), (v, wv)):
        assert got.shape == want.shape and got.dtype == dtype
        assert torch.equal(got.cpu(), torch.from_numpy(want).to(dtype))  # exact: 8-bit values times powers of two


def test_read_scales_that_are_no_powers_of_two():
    cache = filled(3, 2, 16, 32, E4M3, seed=3)
    cache = cache._replace(k_scale=torch.rand(3, 2, generator=gen(1)) + 0.1, v_scale=torch.rand(3, 2, generator=gen(2)))
    table = table_of(1, 3, 3, seed=1)
    lengths = torch.tensor([48], dtype=torch.int32)
    k, v = native.kv8_read(*to_gpu(cache), table.to(DEV), lengths.to(DEV), 48, dtype=F32)
    for got, want in zip((k, v), plain.read(cache, table, lengths, 48)):
        assert np.all(np.abs(got.cpu().numpy() - want) <= 2.0 ** -24 * np.abs(want))


def test_read_nothing():
    cache = to_gpu(filled(2, 2, 16, 32, E4M3, seed=1))
    table = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    lengths = torch.full((2,), 9, dtype=torch.int32, device=DEV)
    assert native.kv8_read(*cache, table, lengths, 0)[0].shape == (2, 2, 0, 32)
    assert native.kv8_read(*cache, table[:0], lengths[:0], 5)[0].shape == (0, 2, 5, 32)
    assert not native.kv8_read(*cache, table[:, :0], lengths, 5)[1].any()
    empty = to_gpu(filled(0, 2, 16, 32, E4M3, seed=1))
    assert not native.kv8_read(*empty, table, lengths, 5)[0].any()


# ---------------------------------------------------------------------------
# attention over all tokens
# ---------------------------------------------------------------------------
def attend_case(B, Q, H, G, D, page, lens, fmt, dtype, seed, stale=None, squeeze=True):
    blocks = max(1, -(-max(max(lens), 1) // page))
    pages = B * blocks + 1
    cache = filled(pages, H, page, D, fmt, seed=seed)
    table = table_of(B, blocks, pages, seed=seed + 1)
    q = torch.randn((B, H * G, D) if Q == 1 and squeeze else (B, Q, H * G, D), generator=gen(seed + 2)).to(dtype)
    lengths = torch.tensor(lens, dtype=torch.int32)
    dirty = cache
    if stale is not None:  # what lies behind the lengths must not matter
        dirty = kv8_layout.Kv8Cache(*(t.clone() for t in cache))
        kb, vb = dirty.k_cache.view(torch.uint8), dirty.v_cache.view(torch.uint8)
        used = set()
        for b in range(B):
            for j in range(blocks):
                p, n = int(table[b, j]), min(max(int(lens[b]) - j * page, 0), page)
                used.add(p)
                kb[p, :, n:] = stale
                rows = vb[p].permute(0, 1, 3, 2).reshape(H, page, D).clone()
                rows[:, n:] = stale
                vb[p] = rows.view(H, page // 16, 16, D).permute(0, 1, 3, 2)
                if n == 0:
                    dirty.k_scale[p], dirty.v_scale[p] = float("nan"), float("inf")
    return q, cache, dirty, table, lengths


def check_attend(q, cache, dirty, table, lengths, **kw):
    got = native.kv8_decode_forward(q.to(DEV), *to_gpu(dirty), table.to(DEV), lengths.to(DEV), **kw)
    assert got.shape == q.shape and got.dtype == q.dtype
    want, mass, size = plain.attend(q, cache, table, lengths, scale=kw.get("softmax_scale"))
    close(got, want, mass, size, int(lengths.max()), peak_of(cache))
    return got


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attend_types_and_head_sizes(fmt, dtype, D):
    check_attend(*attend_case(3, 1, 2, 2, D, 32, (0, 1, 83), fmt, dtype, seed=D, stale=0x7f))


@pytest.mark.parametrize("page", [16, 48, 64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attend_lengths_around_every_border(page, dtype):
    lens = (1, 15, 16, 17, 31, 33, 47, 48, 49, 63, 64, 65, 127, 129, 255, 257, 320, 0)
    check_attend(*attend_case(len(lens), 1, 1, 1, 64, page, lens, E4M3, dtype, seed=page, stale=0xff))


@pytest.mark.parametrize("Q,G", [(1, 3), (1, 5), (1, 8), (1, 16), (1, 20), (1, 64), (2, 1), (3, 5), (4, 4), (8, 2), (17, 1),
                                 (33, 3), (70, 1)])
@pytest.mark.parametrize("fmt,dtype", [(E4M3, BF16), (INT8, F16), (E4M3, F32)])
def test_attend_groups_and_several_queries(Q, G, fmt, dtype):
    """Grouped heads, several query tokens (causal among themselves), sequences
    shorter than the queries, empty ones."""
    check_attend(*attend_case(4, Q, 2, G, 64, 16, (0, 2, Q, 90), fmt, dtype, seed=Q * 64 + G, stale=0x7f))


def test_attend_one_query_given_with_and_without_its_axis():
    q, cache, dirty, table, lengths = attend_case(2, 1, 2, 2, 64, 16, (5, 40), E4M3, BF16, seed=4)
    args = (*to_gpu(cache), table.to(DEV), lengths.to(DEV))
    a = native.kv8_decode_forward(q.to(DEV), *args)
    b = native.kv8_decode_forward(q.to(DEV).unsqueeze(1), *args)
    assert torch.equal(a, b.squeeze(1))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attend_long_context_against_a_device_reference(dtype):
    """Thousands of tokens (many parts, ragged), against fp64 on the device."""
    B, H, G, D, page = 5, 2, 4, 128, 64
    lens = (20000, 1, 7777, 0, 12345)
    blocks = -(-max(lens) // page)
    pages = B * blocks
    cache = to_gpu(filled(pages, H, page, D, E4M3, seed=1, spread=1))
    table = table_of(B, blocks, pages, seed=2).to(DEV)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = torch.randn(B, H * G, D, generator=gen(3)).to(dtype).to(DEV)
    got = native.kv8_decode_forward(q, *cache, table, lengths)
    k, v = native.kv8_read(*cache, table, lengths, max(lens), dtype=F32)
    for b in range(B):
        n = lens[b]
        if n == 0:
            assert not got[b].any()
            continue
        kb, vb, qb = (t.double().cpu().numpy() for t in (k[b, :, :n], v[b, :, :n], q[b].view(H, G, D)))
        for h in range(H):
            for g in range(G):
                want, mass, size = plain._softmax_v(qb[h, g], list(kb[h]), list(vb[h]), D ** -0.5)
                close(got[b, h * G + g], want, mass, np.float64(size), n, peak_of(cache))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_attend_sharp_flat_and_far_scores(dtype):
    """One token far above the rest; all alike; all far below zero; scales of
    pages far apart."""
    B, H, D, page = 4, 1, 64, 16
    lens = (100, 100, 100, 100)
    q, cache, _, table, lengths = attend_case(B, 1, H, 1, D, page, lens, E4M3, dtype, seed=8)
    kb = cache.k_cache.view(torch.uint8)
    kb[int(table[0, 3]), 0, 5] = torch.where(q[0, 0].float() > 0, 0x70, 0xf0).to(torch.uint8)
    for j in range(7):
        kb[int(table[1, j])] = 0
        kb[int(table[2, j]), 0] = torch.where(q[2, 0].float() > 0, 0xf0, 0x70).to(torch.uint8)
        cache.v_scale[int(table[3, j])] = 2.0 ** (6 * j - 20)
        cache.k_scale[int(table[2, j])] = 1.0
    check_attend(q, cache, cache, table, lengths)
    check_attend(q, cache, cache, table, lengths, softmax_scale=0.0)
    check_attend(q, cache, cache, table, lengths, softmax_scale=-0.2)


def test_attend_large_and_small_queries():
    """q far from 1 in magnitude (beyond what f16 holds), zero rows; scores stay moderate by the scale."""
    q, cache, _, table, lengths = attend_case(5, 1, 1, 2, 96, 32, (70,) * 5, E4M3, BF16, seed=12)
    for b, e in enumerate((100, -100, 0, 20, -30)):
        q[b] = (q[b].float() * 2.0 ** e).to(BF16)
    q[2] = 0
    for b, e in enumerate((100, -100, 0, 20, -30)):
        check_attend(q[b : b + 1], cache, cache, table[b : b + 1], lengths[b : b + 1], softmax_scale=2.0 ** (-e - 3))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attend_queries_whose_products_pass_fp32(dtype):
    """q near the type's largest value over pages of tiny keys: the scores are moderate, q times a byte is not."""
    q, cache, _, table, lengths = attend_case(2, 1, 2, 2, 64, 32, (70, 33), E4M3, dtype, seed=13)
    cache.k_scale.fill_(2.0 ** -120)
    q = (q.float().clamp(-3, 3) * 2.0 ** 122).to(dtype)
    check_attend(q, cache, cache, table, lengths, softmax_scale=2.0 ** -9)


@pytest.mark.parametrize("Q,G", [(1, 1), (1, 40), (5, 9), (30, 3), (70, 2)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_attend_v_scales_far_apart(Q, G, dtype):
    """Every page weighs alike, their V differ: some all zeros (the least scale),
    some far larger, some smaller.  The softmax's sum must count them all."""
    lens = (330, 96 + Q, 320, 200, 17 + Q)
    q, cache, _, table, lengths = attend_case(5, Q, 1, G, 64, 16, lens, E4M3, dtype, seed=Q + 3 * G)
    cache.k_scale.mul_(2.0 ** -6)
    cache.v_scale.fill_(2.0 ** -8)
    for j in range(table.shape[1]):
        if j % 3 == 1:
            for b in (0, 1, 4):  # zeros among others
                cache.v_cache.view(torch.uint8)[int(table[b, j])] = 0
                cache.v_scale[int(table[b, j])] = kv8_layout.LEAST_SCALE
        cache.v_scale[int(table[2, j])] = 2.0 ** ((j % 5 - 2) * 7 - 8)
        if j > 7:
            cache.v_scale[int(table[3, j])] = 2.0 ** -70
    for b in range(5):
        row = slice(b, b + 1)
        check_attend(q[row], cache, cache, table[row], lengths[row])
    check_attend(q, cache, cache, table, lengths)


@pytest.mark.parametrize("dtype,G", [(BF16, 3), (F32, 2), (BF16, 80)])
def test_attend_scales_that_are_no_powers_of_two(dtype, G):
    q, cache, _, table, lengths = attend_case(3, 1, 2, G, 64, 16, (70, 300, 16), E4M3, dtype, seed=17)
    for scale in cache[2:]:
        scale.mul_(0.6 + torch.rand(scale.shape, generator=gen(18)))
    check_attend(q, cache, cache, table, lengths)


def test_attend_a_batch_of_more_sequences_than_lanes():
    """Parts are found by a wavefront 64 sequences at a time."""
    B = 150
    lens = tuple(int(x) for x in torch.randint(0, 1300, (B,), generator=gen(19)))
    for Q, n in ((1, lens), (1, (513,) * B), (35, lens)):
        q, cache, dirty, table, lengths = attend_case(B, Q, 1, 2, 32, 64, n, E4M3, BF16, seed=20)
        got = native.kv8_decode_forward(q.to(DEV), *to_gpu(cache), table.to(DEV), lengths.to(DEV))
        rows = list(range(0, B, 7)) + [63, 64, 65, 127, 128, 149]
        want, mass, size = plain.attend(q[rows], cache, table[rows], lengths[rows])
        close(got[rows], want, mass, size, max(n), peak_of(cache))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("down", [118, 90])
def test_attend_tiny_v(dtype, down):
    q, cache, _, table, lengths = attend_case(2, 3, 2, 5, 64, 16, (70, 300), INT8, dtype, seed=14)
    cache.v_scale.mul_(2.0 ** (8 - down))
    check_attend(q, cache, cache, table, lengths)


@pytest.mark.parametrize("Q,dtype", [(1, BF16), (1, F32), (20, BF16), (70, BF16)])
def test_attend_v_scales_that_change_late_in_a_part(Q, dtype):
    """Parts of more tiles than are looked up at once, V scales far apart from the
    270th tile on: sums begun one way are carried on the other and joined."""
    H, D, page, n = 32, 32, 256, 160000
    pool, blocks = 24, -(-n // page)
    cache = filled(pool, H, page, D, E4M3, seed=15, spread=0)
    cache.k_scale.mul_(2.0 ** -6)
    cache.v_cache.view(torch.uint8)[20:22] = 0
    cache.v_scale[20:22] = kv8_layout.LEAST_SCALE
    cache.v_scale[22:] *= 2.0 ** 20
    table = (torch.arange(blocks) % 20).view(1, blocks).to(torch.int32)
    for tile in range(270, 300, 4):
        table[0, tile // 4] = 20 + tile // 4 % 4
    lengths = torch.tensor([n], dtype=torch.int32)
    q = torch.randn(1, Q, H, D, generator=gen(16)).to(dtype)
    dev = to_gpu(cache)
    got = native.kv8_decode_forward(q.to(DEV), *dev, table.to(DEV), lengths.to(DEV))
    k, v = native.kv8_read(*dev, table.to(DEV), lengths.to(DEV), n, dtype=F32)
    sees = n - Q + 1 + torch.arange(Q, device=DEV)
    hidden = torch.arange(n, device=DEV)[None] >= sees[:, None]
    for h in range(0, H, 5):
        kh, vh, qh = k[0, h].double(), v[0, h].double(), q[0, :, h].to(DEV).double()
        s = qh @ kh.T.contiguous() * D ** -0.5
        p = torch.softmax(s.masked_fill(hidden, -float("inf")), -1)
        size = (qh.abs() @ kh.abs().T.contiguous()).max(-1).values * D ** -0.5
        want, mass = p @ vh, p @ vh.abs()
        close(got[0, :, h], want.cpu().numpy(), mass.cpu().numpy(), size.cpu().numpy(), n, peak_of(cache))


def test_attend_nan_and_infinite_inputs_stay_in_their_row():
    q, cache, _, table, lengths = attend_case(3, 1, 1, 2, 64, 16, (40, 40, 40), E4M3, BF16, seed=6)
    q[0, 1, 3] = float("nan")
    q[1, 0, 5] = float("inf")
    cache.v_cache.view(torch.uint8)[int(table[2, 1]), 0, 0, 7, 2] = 0x7f  # a NaN that was stored
    got = native.kv8_decode_forward(q.to(DEV), *to_gpu(cache), table.to(DEV), lengths.to(DEV)).cpu()
    assert got[0, 1].isnan().all() and got[1, 0].isnan().all() and got[2, :, 7].isnan().all()
    clean = got.clone()
    clean[0, 1], clean[1, 0], clean[2, :, 7] = 0, 0, 0
    assert clean.isfinite().all()
    want, mass, size = plain.attend(q[0:1, 0:1], cache, table[0:1], lengths[0:1])
    close(got[0:1, 0:1], want, mass, size, 40, peak_of(cache))


@pytest.mark.parametrize("Q,G,D", [(3, 2, 64), (20, 1, 96), (70, 1, 64), (70, 3, 128), (90, 4, 192), (150, 2, 32)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attend_nan_in_a_later_query_s_token_stays_with_its_seers(Q, G, D, dtype):
    """V of a token that only the later queries of the call see is NaN (and K of
    another): the earlier queries are as if it were not there."""
    n = Q + 40
    q, cache, _, table, lengths = attend_case(2, Q, 1, G, D, 16, (n, n), E4M3, dtype, seed=Q)
    vb, kb = cache.v_cache.view(torch.uint8), cache.k_cache.view(torch.uint8)
    at_v, at_k = n - Q // 2, n - 1  # seen from query Q - Q // 2 on, and by the last
    vb[int(table[0, at_v // 16]), 0, 0, 5, at_v % 16] = 0xff
    vb[int(table[0, at_v // 16]), 0, 0, D - 1, at_v % 16] = 0x7f
    kb[int(table[1, at_k // 16]), 0, at_k % 16, 3] = 0x7f
    got = native.kv8_decode_forward(q.to(DEV), *to_gpu(cache), table.to(DEV), lengths.to(DEV))
    want, mass, size = plain.attend(q, cache, table, lengths)
    first = at_v - (n - Q)
    assert np.isnan(want[0, first:, :, 5]).all() and np.isnan(want[1, -1]).all() and np.isfinite(want[0, :first]).all()
    assert np.array_equal(np.isnan(got.float().cpu().numpy()), np.isnan(want))
    fine = torch.from_numpy(np.isnan(want))
    got, want, mass = got.cpu().masked_fill(fine, 0), np.nan_to_num(want), np.nan_to_num(mass)
    close(got, want, mass, np.nan_to_num(size), n, peak_of(cache))


def test_attend_pages_outside_the_pool_are_skipped():
    q, cache, _, table, lengths = attend_case(3, 1, 2, 1, 64, 16, (60, 60, 30), INT8, F16, seed=7)
    table[0, 1], table[1, 0], table[1, 1], table[1, 2], table[1, 3] = -7, -1, 10 ** 6, -2 ** 31, 2 ** 31 - 1
    check_attend(q, cache, cache, table, lengths)


def test_attend_lengths_outside_the_table():
    q, cache, _, table, lengths = attend_case(3, 2, 2, 1, 64, 16, (40, 40, 40), E4M3, BF16, seed=7)
    lengths = torch.tensor([-5, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    want, mass, size = plain.attend(q, cache, table, lengths)
    got = native.kv8_decode_forward(q.to(DEV), *to_gpu(cache), table.to(DEV), lengths.to(DEV))
    close(got, want, mass, size, 48, peak_of(cache))
    assert not got[0].any() and not got[2].any()


def test_attend_a_table_with_wider_rows():
    q, cache, dirty, table, lengths = attend_case(3, 1, 2, 1, 64, 16, (40, 9, 33), E4M3, BF16, seed=17)
    wide = torch.full((3, 11), -1, dtype=torch.int32)
    wide[:, 4 : 4 + table.shape[1]] = table
    got = native.kv8_decode_forward(q.to(DEV), *to_gpu(cache), wide.to(DEV)[:, 4 : 4 + table.shape[1]], lengths.to(DEV))
    assert torch.equal(got, native.kv8_decode_forward(q.to(DEV), *to_gpu(cache), table.to(DEV), lengths.to(DEV)))


def test_attend_nothing():
    cache = to_gpu(filled(2, 2, 16, 32, E4M3, seed=1))
    table = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    lengths = torch.full((2,), 9, dtype=torch.int32, device=DEV)
    q = torch.ones(2, 3, 4, 32, dtype=BF16, device=DEV)
    assert native.kv8_decode_forward(q[:0], *cache, table[:0], lengths[:0]).shape == (0, 3, 4, 32)
    assert native.kv8_decode_forward(q[:, :0].contiguous(), *cache, table, lengths).shape == (2, 0, 4, 32)
    assert not native.kv8_decode_forward(q, *cache, table[:, :0], lengths).any()
    assert not native.kv8_decode_forward(q, *to_gpu(filled(0, 2, 16, 32, E4M3, seed=1)), table, lengths).any()


def test_attend_pool_beyond_32_bit_offsets():
    """Pages whose bytes lie past 4 GiB."""
    H, page, D = 8, 256, 256
    pages = (1 << 32) // (H * page * D) + 5
    cache = kv8_layout.empty_cache(pages, H, page, D, device=DEV)
    table = torch.tensor([[pages - 1, pages - 3, 0]], dtype=torch.int32)
    g = gen(5)
    k, v = (torch.randn(1, H, 600, D, generator=g).to(BF16) for _ in range(2))
    zero, n = torch.zeros(1, dtype=torch.int32), torch.tensor([600], dtype=torch.int32)
    native.kv8_write(k.to(DEV), v.to(DEV), *cache, table.to(DEV), zero.to(DEV))
    q = torch.randn(1, H, D, generator=g).to(BF16)
    got = native.kv8_decode_forward(q.to(DEV), *cache, table.to(DEV), n.to(DEV))
    ids = torch.tensor([[[0, 9, 5, 8]]], dtype=torch.int32).expand(1, H, 4).contiguous()
    got_csa = native.kv8_csa_decode_forward(q.to(DEV), *cache, table.to(DEV), n.to(DEV), ids.to(DEV), 64)
    # the same three pages in a small pool
    at = table[0].long().to(DEV)
    small = tuple(t.view(torch.uint8)[at].view(t.dtype) if t.dtype == E4M3 else t[at] for t in cache)
    near = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV)
    assert torch.equal(got, native.kv8_decode_forward(q.to(DEV), *small, near, n.to(DEV)))
    assert torch.equal(got_csa, native.kv8_csa_decode_forward(q.to(DEV), *small, near, n.to(DEV), ids.to(DEV), 64))
    for a, b in zip(native.kv8_read(*cache, table.to(DEV), n.to(DEV), 600), native.kv8_read(*small, near, n.to(DEV), 600)):
        assert torch.equal(a, b) and a.any()


# ---------------------------------------------------------------------------
# attention over listed chunks
# ---------------------------------------------------------------------------
def check_csa(q, cache, dirty, table, lengths, chunks, chunk):
    got = native.kv8_csa_decode_forward(q.to(DEV), *to_gpu(dirty), table.to(DEV), lengths.to(DEV), chunks.to(DEV), chunk)
    want, mass, size = plain.attend(q, cache, table, lengths, chunks=chunks.numpy(), chunk_size=chunk)
    close(got, want, mass, size, chunks.shape[2] * chunk, peak_of(cache))
    return got


@pytest.mark.parametrize("chunk,top_k", [(1, 5), (7, 9), (16, 1), (16, 13), (20, 3), (48, 4), (64, 1), (64, 8), (100, 3),
                                         (130, 2), (1000, 2)])
@pytest.mark.parametrize("fmt,dtype,page", [(E4M3, BF16, 64), (INT8, F16, 16), (E4M3, F32, 48)])
def test_csa_chunk_sizes(chunk, top_k, fmt, dtype, page):
    """Chunks that begin and end anywhere in a page; a last chunk cut by the length."""
    B, H, G, D = 2, 2, 2, 64
    q, cache, dirty, table, lengths = attend_case(B, 1, H, G, D, page, (301, 290), fmt, dtype, seed=chunk, stale=0x7f)
    C = -(-301 // chunk)
    chunks = torch.stack([torch.randperm(C, generator=gen(chunk + i))[:top_k] for i in range(B * H)])
    chunks = chunks.view(B, H, -1).to(torch.int32 if chunk % 2 else torch.int64)
    check_csa(q, cache, dirty, table, lengths, chunks, chunk)


@pytest.mark.parametrize("G", [17, 40, 100])
@pytest.mark.parametrize("fmt,dtype", [(E4M3, BF16), (INT8, F16), (E4M3, F32)])
def test_csa_many_heads_share_a_list(G, fmt, dtype):
    q, cache, dirty, table, lengths = attend_case(2, 1, 1, G, 96, 48, (301, 77), fmt, dtype, seed=G, stale=0x7f)
    chunks = torch.tensor([[[3, 0, -1, 9, 4, 4]], [[1, 0, 2, 3, 0, 7]]], dtype=torch.int32)
    check_csa(q, cache, dirty, table, lengths, chunks, 36)


@pytest.mark.parametrize("G", [1, 20, 70])
def test_csa_of_pages_of_zeros_among_others(G):
    q, cache, _, table, lengths = attend_case(2, 1, 1, G, 64, 16, (300, 77), E4M3, BF16, seed=G)
    cache.k_scale.mul_(2.0 ** -6)
    for b, j in ((0, 1), (0, 4), (1, 0), (1, 2)):
        cache.v_cache.view(torch.uint8)[int(table[b, j])] = 0
        cache.v_scale[int(table[b, j])] = kv8_layout.LEAST_SCALE
    chunks = torch.tensor([[[3, 0, 1, 2, 5]], [[1, 0, 2, 2, -1]]], dtype=torch.int32)
    check_csa(q, cache, cache, table, lengths, chunks, 32)


@pytest.mark.parametrize("D", [32, 64, 96, 160, 192, 224, 256])
@pytest.mark.parametrize("fmt,dtype", [(E4M3, BF16), (INT8, F16)])
def test_attend_many_rows_of_every_head_size(D, fmt, dtype):
    """More rows than a workgroup of the kernel for many takes, a few of the last one."""
    check_attend(*attend_case(3, 45, 1, 3, D, 32, (0, 44, 130), fmt, dtype, seed=D + 1, stale=0x7f))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_attend_many_rows_over_many_tiles(dtype):
    """A prompt chunk over thousands of tokens: several lookups of pages, several
    parts, against fp64 on the device."""
    B, Q, H, G, D, page = 2, 70, 1, 2, 64, 64
    lens = (9000, 4161)
    blocks = -(-max(lens) // page)
    cache = to_gpu(filled(B * blocks, H, page, D, E4M3, seed=1, spread=1))
    table = table_of(B, blocks, B * blocks, seed=2).to(DEV)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = torch.randn(B, Q, H * G, D, generator=gen(3)).to(dtype).to(DEV)
    got = native.kv8_decode_forward(q, *cache, table, lengths)
    k, v = native.kv8_read(*cache, table, lengths, max(lens), dtype=F32)
    for b in range(B):
        for i in (0, 1, 37, Q - 1):
            n = lens[b] - Q + 1 + i
            kb, vb, qb = (t.double().cpu().numpy() for t in (k[b, 0, :n], v[b, 0, :n], q[b, i]))
            for h in range(G):
                want, mass, size = plain._softmax_v(qb[h], list(kb), list(vb), D ** -0.5)
                close(got[b, i, h], want, mass, np.float64(size), n, peak_of(cache))


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_csa_ids_that_are_negative_repeated_or_too_large(index):
    B, H, G, D, page, chunk = 6, 1, 3, 64, 16, 24
    q, cache, dirty, table, lengths = attend_case(B, 1, H, G, D, page, (100, 100, 100, 0, 100, 30), E4M3, BF16, seed=3,
                                                  stale=0x7f)
    big = torch.iinfo(index).max
    rows = [[0, -1, 2, -5], [3, 3, 3, 1], [-1, -1, -2, -3], [0, 1, 2, 3], [4, big, 5, big // chunk], [0, 1, 1, 2]]
    chunks = torch.tensor(rows, dtype=index).view(B, H, 4)
    got = check_csa(q, cache, dirty, table, lengths, chunks, chunk)
    assert not got[2].any() and not got[3].any()


def test_csa_no_chunks_and_bad_pages():
    q, cache, _, table, lengths = attend_case(2, 1, 2, 1, 64, 16, (100, 100), E4M3, BF16, seed=3)
    none = torch.zeros(2, 2, 0, dtype=torch.int32)
    assert not check_csa(q, cache, cache, table, lengths, none, 16).any()
    table[0, 2], table[1, 0] = -1, 10 ** 6
    chunks = torch.tensor([[[2, 1], [0, 2]], [[0, 0], [3, 0]]], dtype=torch.int32)
    check_csa(q, cache, cache, table, lengths, chunks, 16)


def test_csa_of_every_chunk_is_the_dense_attention():
    q, cache, _, table, lengths = attend_case(3, 1, 2, 2, 128, 64, (640, 501, 77), E4M3, BF16, seed=5)
    chunks = torch.arange(10, dtype=torch.int32).expand(3, 2, 10).contiguous()
    got = check_csa(q, cache, cache, table, lengths, chunks, 64).float()
    want = native.kv8_decode_forward(q.to(DEV), *to_gpu(cache), table.to(DEV), lengths.to(DEV)).float()
    assert torch.all((got - want).abs() <= 2 * 2.0 ** -8 * want.abs() + 2.0 ** -9 * want.abs().max())


# ---------------------------------------------------------------------------
# together, in graphs, on streams
# ---------------------------------------------------------------------------
def test_prompt_and_decode_steps_run_together():
    """A prompt written, read back for its chunk summaries, chunks selected and
    attended to; then tokens appended one at a time and attended to, against the
    ops over the read-back 32-bit cache."""
    B, H, D, page, chunk, S = 2, 4, 128, 64, 64, 1024
    cache = kv8_layout.empty_cache(B * 18, H, page, D, device=DEV)
    table = table_of(B, 18, B * 18, seed=1).to(DEV)
    g = gen(2)
    qkv = torch.randn(B, S, 3, H, D, generator=g).to(BF16).to(DEV)
    start = torch.zeros(B, dtype=torch.int32, device=DEV)
    extension.kv8_write(qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2), *cache, table, start)
    lengths = start + S
    k, v = extension.kv8_read(*cache, table, lengths, S, dtype=F32)
    summary = native.csa_chunk_summary(k, chunk)
    q = qkv[:, -1, 0].contiguous()
    ids = extension.csa_select_topk(q, summary, 8)
    got = extension.kv8_csa_decode_forward(q, *cache, table, lengths, ids, chunk)
    want = extension.csa_decode_forward(q.float(), k, v, ids, chunk)
    # both sides: a weight's rounding to 11 bits here, and half a bf16 step of the result
    assert torch.all((got.float() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * v.abs().max())
    for t in range(3):
        new = torch.randn(B, 3, H, D, generator=g).to(BF16).to(DEV)
        extension.kv8_write(new[:, 1].unsqueeze(2), new[:, 2].unsqueeze(2), *cache, table, lengths)
        lengths = lengths + 1
        got = extension.kv8_decode_forward(new[:, 0].contiguous(), *cache, table, lengths)
        k, v = extension.kv8_read(*cache, table, lengths, S + t + 1, dtype=F32)
        one = torch.zeros(B, H, 1, dtype=torch.int32, device=DEV)
        want = extension.csa_decode_forward(new[:, 0].float().contiguous(), k, v, one, S + t + 1)
        assert torch.all((got.float() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * v.abs().max())


def test_captured_steps_replay_to_the_eager_results():
    """Two graphs (a decode step of write and attend; a sparse read of the same
    cache) captured on one stream, replayed in turn and on two streams, between
    eager calls: each replay gives what the eager calls give."""
    B, H, G, D, page = 3, 2, 4, 128, 32
    cache = kv8_layout.empty_cache(B * 64, H, page, D, dtype=INT8, device=DEV)
    eager = tuple(t.clone() for t in cache)
    table = table_of(B, 64, B * 64, seed=4).to(DEV)
    x = torch.randn(2, B, H, 1900, D, generator=gen(9)).to(F16).to(DEV)
    zero = torch.zeros(B, dtype=torch.int32, device=DEV)
    for c in (cache, eager):
        native.kv8_write(x[0], x[1], *c, table, zero)
    lengths = torch.tensor([1900, 700, 3], dtype=torch.int32, device=DEV)
    q = torch.empty(B, H * G, D, dtype=F16, device=DEV)
    new = torch.empty(2, B, H, 1, D, dtype=F16, device=DEV)
    ids = torch.randint(0, 30, (B, H, 16), generator=gen(1)).to(torch.int32).to(DEV)

    def step(c, n):
        native.kv8_write(new[0], new[1], *c, table, n)
        n.add_(1)
        return native.kv8_decode_forward(q, *c, table, n)

    def sparse(c, n):
        return native.kv8_csa_decode_forward(q, *c, table, n, ids, 64)

    q.normal_(), new.normal_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    n_graph, n_eager = lengths.clone(), lengths.clone()
    graphs = []
    with torch.cuda.stream(s):
        for f in (step, sparse):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                out = f(cache, n_graph)
            graphs.append((graph, out))
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for _ in range(4):
        q.normal_(), new.normal_()
        want = step(eager, n_eager).clone()
        torch.cuda.synchronize()
        graphs[0][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want)
        want_sparse = sparse(eager, n_eager)
        torch.cuda.synchronize()
        # both at once: the dense attention of the next token and the sparse one of this cache
        with torch.cuda.stream(other):
            graphs[1][0].replay()
        again = native.kv8_decode_forward(q, *cache, table, n_graph)
        torch.cuda.synchronize()
        assert torch.equal(graphs[1][1], want_sparse) and torch.equal(again, want)
        for a, b in zip(cache, eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_results_do_not_change_from_call_to_call():
    q, cache, _, table, lengths = attend_case(3, 2, 2, 4, 128, 64, (5000, 900, 4097), E4M3, BF16, seed=21)
    args = (q.to(DEV), *to_gpu(cache), table.to(DEV), lengths.to(DEV))
    first = native.kv8_decode_forward(*args)
    for _ in range(3):
        assert torch.equal(first, native.kv8_decode_forward(*args))


def test_calls_of_two_host_threads_on_one_stream_and_on_two():
    q, cache, _, table, lengths = attend_case(3, 2, 2, 4, 64, 64, (5000, 900, 4097), E4M3, BF16, seed=22)
    args = (*to_gpu(cache), table.to(DEV), lengths.to(DEV))
    qs = [q.to(DEV), (q * 0.5).to(DEV)]
    want = [native.kv8_decode_forward(x, *args) for x in qs]
    torch.cuda.synchronize()
    for streams in ([torch.cuda.current_stream()] * 2, [torch.cuda.Stream(), torch.cuda.Stream()]):
        got = [[], []]

        def calls(i):
            with torch.cuda.stream(streams[i]):
                for _ in range(20):
                    got[i].append(native.kv8_decode_forward(qs[i], *args))
                streams[i].synchronize()

        threads = [threading.Thread(target=calls, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for i in range(2):
            assert len(got[i]) == 20 and all(torch.equal(x, want[i]) for x in got[i])


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals():
    cache = to_gpu(filled(4, 2, 16, 64, E4M3, seed=1))
    k, v, ks, vs = cache
    table = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    n = torch.ones(2, dtype=torch.int32, device=DEV)
    q = torch.zeros(2, 4, 64, dtype=BF16, device=DEV)
    x = torch.zeros(2, 2, 3, 64, dtype=BF16, device=DEV)

    def refused(match, f, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            f(*args, **kw)

    att = native.kv8_decode_forward
    refused("CUDA tensors", att, q, k.cpu(), v, ks, vs, table, n)
    refused("k_cache must be \\[", att, q, k[0], v, ks, vs, table, n)
    refused("must be contiguous", att, q, k.transpose(1, 2), v, ks, vs, table, n)
    refused("float8_e4m3fn or int8", att, q, k.view(torch.uint8), v.view(torch.uint8), ks, vs, table, n)
    refused("dtype must match", att, q, k, v.view(INT8), ks, vs, table, n)
    refused("v_cache must be", att, q, k, v.view(4, 2, 64, 1, 16), ks, vs, table, n)
    refused("scales must be", att, q, k, v, ks.double(), vs, table, n)
    refused("scales must be", att, q, k, v, ks, vs[:, :1], table, n)
    refused("block_table must be int32", att, q, k, v, ks, vs, table.long(), n)
    refused("rows must be contiguous", att, q, k, v, ks, vs, table.t(), n)
    refused("one row per sequence", att, q, k, v, ks, vs, table[:1], n[:1])
    refused("lengths must be", att, q, k, v, ks, vs, table, n.long())
    refused("lengths must be", att, q, k, v, ks, vs, table, n[:1])
    refused("lengths must be", att, q, k, v, ks, vs, table, None)
    refused("q must be contiguous", att, q.transpose(0, 1), k, v, ks, vs, table, n)
    refused("multiple of the cache's heads", att, q[:, :3].contiguous(), k, v, ks, vs, table, n)
    refused("cache's head_dim", att, q[..., :32].contiguous(), k, v, ks, vs, table, n)
    refused("unsupported dtype", att, q.double(), k, v, ks, vs, table, n)
    refused("q must be \\[", att, q[0], k, v, ks, vs, table, n)
    odd = torch.zeros(q.numel() + 1, dtype=BF16, device=DEV)[1:].view(q.shape)
    refused("16-byte aligned", att, odd, k, v, ks, vs, table, n)
    refused("rows overlap", att, q, k, v, ks, vs, table[:1].expand(2, 2), n)
    csa = native.kv8_csa_decode_forward
    ids = torch.zeros(2, 2, 1, dtype=torch.int32, device=DEV)
    refused("q must be \\[", csa, q.unsqueeze(1), k, v, ks, vs, table, n, ids, 16)
    refused("chunk_size must be positive", csa, q, k, v, ks, vs, table, n, ids, 0)
    refused("int32 or int64", csa, q, k, v, ks, vs, table, n, ids.float(), 16)
    refused("\\[batch, kv_heads, top_k\\]", csa, q, k, v, ks, vs, table, n, ids[:, :1].contiguous(), 16)
    wr = native.kv8_write
    refused("new_tokens, head_dim\\]", wr, x[0], x[0], *cache, table, n)
    refused("float32, float16 or bfloat16", wr, x.double(), x.double(), *cache, table, n)
    refused("float32, float16 or bfloat16", wr, x, x.half(), *cache, table, n)
    refused("contiguous in head_dim", wr, x.transpose(2, 3).contiguous().transpose(2, 3), x, *cache, table, n)
    refused("cache's heads", wr, x[:, :1], x[:, :1], *cache, table, n)
    refused("start must be", wr, x, x, *cache, table, n.long())
    refused("counts must be", wr, x, x, *cache, table, n, counts=n[:1])
    rd = native.kv8_read
    refused("unsupported dtype", rd, *cache, table, n, 4, dtype=torch.float64)
    refused("non-negative", rd, *cache, table, n, -1)
    refused("start must be", rd, *cache, table, n, 4, start=n.long())
    odd = torch.zeros(k.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(E4M3).view(k.shape)
    refused("16-byte aligned", att, q, odd, v, ks, vs, table, n)
    for D in (48, 288):
        refused("multiple of 32", att, q, *to_gpu(kv8_layout.Kv8Cache(*_shaped(16, D))), table, n)
    for page in (8, 272):
        refused("multiple of 16", att, q, *to_gpu(kv8_layout.Kv8Cache(*_shaped(page, 64))), table, n)
    for dtype, page, D in ((torch.uint8, 16, 64), (E4M3, 8, 64), (E4M3, 16, 48)):
        with pytest.raises(ValueError):
            kv8_layout.empty_cache(1, 1, page, D, dtype=dtype)


def _shaped(page, D):
    k = torch.zeros(4, 2, page, D, dtype=torch.uint8).view(E4M3)
    return k, torch.zeros(4, 2, max(page // 16, 1), D, 16, dtype=torch.uint8).view(E4M3), torch.ones(4, 2), torch.ones(4, 2)
