"""Precision of paged attention (x_attn_paged) where weights span many powers of two, where sums run over long contexts,
and where a lower term of a probability counts. Bounds are relative to the output, or to the values' mean size.
"""
import copy
import ctypes as C

import numpy as np
import pytest
import torch

import attnref as ref


def _run(lib, b, q, group, scale, bf16):
    dtype = torch.bfloat16 if bf16 else torch.float32
    width = b.heads * group * b.dim
    out, dq = ref.up(torch.full((b.tokens, width), 5.0, dtype=dtype)), ref.up(q)
    rc = lib.qwn_x_attn_paged(C.byref(b.cache), C.byref(b.batch), dq.ptr, b.heads * group, scale, out.ptr, width, int(bf16))
    assert rc == 0
    lib.tq_sync()
    assert lib.tq_last_error() == 0
    return ref.down(out, dtype, (b.tokens, width))


# What fp32 outputs may lose in sums over keys, in the values' mean size, whatever the length. The tensor core cuts an
# fp32 sum off, twice in a step of 16 keys (8 and 8), by 2^-23 of the sum so far each time at most; of a sum that grows
# evenly, n cuts take n x 2^-24. Sums have 64 steps at most before they are added to an fp32 sum.
SUMS = 128 * 2.0 ** -24


def _shared(b, count):
    """The batch's one request `count` times over the same pages (they are only read); the batch with it once."""
    once = copy.copy(b)
    new, total = b.lens[0]
    b.lens = b.lens * count
    b.start = (np.arange(count + 1) * new).astype(np.int32)
    b.kv_len = np.full(count, total, np.int32)
    b.table = np.repeat(b.table, count, 0)
    b.tokens = count * new
    return once


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16_cache", "e4m3_cache"])
@pytest.mark.parametrize("depth", [16, 20, 24])
@pytest.mark.parametrize("new,dim", [(1, 64), (1, 128), (1, 256), (100, 64), (100, 128), (100, 256)])
def test_one_key_far_above_the_rest(lib, new, dim, depth, e4m3, bf16):
    """The first key has nearly all the weight and the value 0; 8191 others, some 2^-depth of it each, carry the result
    with values of one sign. Many requests share the pages, so that a CTA takes all keys of one.

    Relative to the output, fp32: a score of size depth (in base 2) has a factor of three roundings and is itself rounded
    beside the maximum, 4 depth ln 2 roundings of 2^-24; the exponentials, 2^-22 above and below; the sums' steps (see
    SUMS). Two fp16 terms of an e4m3 cache's probabilities lose 2^-40 of the largest weight, above 16 rows 2^-36: 2^depth
    as much of one of these, whose random part may put it 2^-1 lower. bf16: a rounding of a probability, 2^-9
    (fp16 for e4m3: 2^-12, or where it ends), averaged over thousands but taken whole here, the exponentials' 7.5e-5, a
    sum of all 8192 keys in steps of 16, and the store's 2^-9."""
    total = 8192 + new - 1
    b = ref.Batch([(new, total)], 64, 1, dim, e4m3, seed=depth + dim)
    g, unit = b.gen, 16.0 if e4m3 else 1.0               # pools hold k / k_scale
    p = np.arange(total)
    page, slot = torch.from_numpy(b.table[0, p // 64]).long(), p % 64
    k0 = torch.randn(total, generator=g) * 0.25
    k0[0] = 8.0
    k = b.k.float()
    k[page, 0, slot, 0] = k0 * unit
    v = b.v.float().abs() * 0.25 + b.v.float().abs().amax() * 0.25
    v[page[0], 0, slot[0]] = 0.0
    b.k.copy_(k.to(b.dtype))
    b.v.copy_(v.to(b.dtype))
    count = 320 if new == 1 else 80
    one = _shared(b, count)
    b.upload()
    q = torch.zeros(b.tokens, 2, dim)
    q[..., 0] = 1.0
    q = q.to(torch.bfloat16)
    scale = float(np.float32(depth * np.log(2.0) / 8.0))
    got = _run(lib, b, q, 2, scale, bf16).double().reshape(count, new, -1)
    want = ref.attention(one, q[:new], 2, scale)
    bound = SUMS + (2.8 * depth + 8) * 2.0 ** -24 + (2.0 ** (depth - (39 if new == 1 else 35)) if e4m3 else 0.0)
    if bf16:
        bound += 2.0 ** -8 + 2.0 ** -13.7 + 1024 * 2.0 ** -24
    off = ((got - want) / want).abs().max().item()
    assert off <= bound, (off, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16_cache", "e4m3_cache"])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_values_of_one_sign_over_long_stretches(lib, dim, new, e4m3):
    """80 requests of 32768 keys (the same pages: they are only read), so that a CTA sums tens of thousands of keys in a
    row, with values around 1 and nearly equal weights.

    The rest, beside the sums' steps (see SUMS): the exponentials' 2^-22, weighted by the values' spread of a tenth, and
    roundings to nearest of some hundred partial sums, 2^-20. All of it in the values' mean size, 1."""
    count, total, group = 80, 32768, 4
    b = ref.Batch([(new, total)], 64, 2, dim, e4m3, seed=dim + new)
    k = (torch.randn(b.k.shape, generator=b.gen) / b.k_scale).to(b.dtype)
    v = ((1.0 + 0.1 * torch.randn(b.v.shape, generator=b.gen)) / b.v_scale).to(b.dtype)
    b.k.copy_(k)
    b.v.copy_(v)
    one = _shared(b, count)
    b.upload()
    q = torch.randn(b.tokens, 2 * group, dim, generator=b.gen).to(torch.bfloat16)
    scale = 0.25 * dim ** -0.5
    got = _run(lib, b, q, group, scale, False).double()
    assert torch.isfinite(got).all()
    bound = SUMS + 2.0 ** -20
    for r in (0, 41, 79):                                # three of the requests in 64 bits
        want = ref.attention(one, q[r * new:(r + 1) * new], group, scale)
        off = (got[r * new:(r + 1) * new] - want).abs().max().item()
        assert off <= bound, (r, off, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16_cache", "e4m3_cache"])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_bf16_outputs_of_long_stretches_lean_nowhere(lib, dim, new, e4m3):
    """131072 keys and more in a row. Each dim's values spread around a mean of its own between 1 and 2, so that outputs lie
    anywhere between two steps of bf16 and their roundings go both ways, but all outputs of a dim lie together (a sum of so
    many keys moves by 3e-4): over `dim` of them the mean of the roundings is 2^-9 / sqrt(3 dim), four times that at most.
    What else is left in the mean is what sums over keys lose: 512 steps of the tensor core, two cuts each (see SUMS), above
    16 rows; up to 16 rows a step per 64 keys, 1536 for a stretch of a request and a half. Probabilities are rounded to
    nearest, and all alike a quarter of a chunk's exponentials, above and below the fraction line."""
    count, total = 160, 131072
    b = ref.Batch([(new, total)], 64, 1, dim, e4m3, seed=dim + new)
    k = (torch.randn(b.k.shape, generator=b.gen) / b.k_scale).to(b.dtype)
    mean = 1.0 + torch.rand(dim, generator=b.gen)
    v = (mean * (1.0 + 0.1 * torch.randn(b.v.shape, generator=b.gen)) / b.v_scale).to(b.dtype)
    b.k.copy_(k)
    b.v.copy_(v)
    one = _shared(b, count)
    b.upload()
    q = torch.randn(b.tokens, 8, dim, generator=b.gen).to(torch.bfloat16)
    scale = 0.25 * dim ** -0.5
    got = _run(lib, b, q, 8, scale, True).double().reshape(count, new, 8 * dim)
    lean = []
    for r in (0, 79, 159):
        want = ref.attention(one, q[r * new:(r + 1) * new], 8, scale)
        lean.append(((got[r] - want) / want).mean().item())
    assert max(abs(x) for x in lean) <= 1536 * 2.0 ** -24 + 4 * 2.0 ** -9 / (3 * dim) ** 0.5, lean


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16_cache", "e4m3_cache"])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_lower_terms_of_probabilities_count(lib, dim, new, e4m3):
    """Nearly equal weights and positive values, 100 keys: what a probability's terms leave out would show whole.

    Two blocks of 64 keys take up to 8 steps of first terms, 16 cuts of 2^-24 (see SUMS), the lower terms' as much at most:
    2^-19; the exponentials' 2^-22, in numerator and denominator. Without the third bf16 term a probability loses 2^-17 on average,
    without the second fp16 one up to 2^-12."""
    b = ref.Batch([(new, 100), (1, 65), (min(new, 3), 17)], 16, 2, dim, e4m3, seed=dim + new)
    v = (b.v.float().abs() * 0.25 + (8.0 if e4m3 else 1.0)).to(b.dtype)
    b.v.copy_(v)
    b.upload()
    q = torch.randn(b.tokens, 6, dim, generator=b.gen).to(torch.bfloat16)
    scale = 0.125 * dim ** -0.5
    got = _run(lib, b, q, 3, scale, False).double()
    want = ref.attention(b, q, 3, scale)
    off = ((got - want) / want).abs().max().item()
    assert off <= 2.0 ** -18.75, (off, 2.0 ** -18.75)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16_cache", "e4m3_cache"])
@pytest.mark.parametrize("growth", [30, 150])
@pytest.mark.parametrize("new,dim", [(1, 128), (20, 64), (20, 128), (20, 256)])
def test_a_maximum_that_keeps_growing(lib, new, dim, growth, e4m3, bf16):
    """Scores grow evenly by 2^growth over 20000 keys, so that the running maximum does so from block to block.

    fp32, relative to the largest value: the sums (see SUMS), and scores' roundings, 4 growth ln 2 of 2^-24 each, above and
    below the fraction line. bf16: the store and the probabilities, 2^-9 each."""
    total, count = 20000, 160
    b = ref.Batch([(new, total)], 64, 1, dim, e4m3, seed=growth + dim)
    p = np.arange(total)
    page, slot = torch.from_numpy(b.table[0, p // 64]).long(), p % 64
    k = b.k.float()
    k[page, 0, slot, 0] = torch.arange(total) / total * 8.0 / b.k_scale
    b.k.copy_(k.to(b.dtype))
    one = _shared(b, count)
    b.upload()
    q = torch.zeros(b.tokens, 2, dim)
    q[..., 0] = 1.0
    q = q.to(torch.bfloat16)
    scale = float(np.float32(growth * np.log(2.0) / 8.0))
    got = _run(lib, b, q, 2, scale, bf16).double().reshape(count, new, -1)
    want = ref.attention(one, q[:new], 2, scale)
    top = b.v.double().abs().max().item() * b.v_scale
    bound = 2.0 ** -8 if bf16 else SUMS + 5.6 * growth * 2.0 ** -24
    off = (got - want).abs().max().item()
    assert off <= top * bound, (off / top, bound)


def _nan_key(lib, new, dim, e4m3, bf16, at):
    """A key of NaN at position `at` of the first request: rows that see it are NaN, the others keep their values."""
    b = ref.Batch([(new, 128 + new), (2, 90)], 16, 1, dim, e4m3, seed=at)
    q = torch.randn(b.tokens, 2, dim, generator=b.gen).to(torch.bfloat16)
    clean = ref.attention(b, q, 2, dim ** -0.5)
    k = b.k.float()
    k[b.table[0, at // 16], 0, at % 16] = float("nan")
    b.k.copy_(k.to(b.dtype))
    b.upload()
    got = _run(lib, b, q, 2, dim ** -0.5, bf16).double()
    sees = torch.zeros(b.tokens, dtype=torch.bool)
    sees[max(0, at - 128):new] = True
    assert torch.isnan(got[sees]).all()
    top = b.v.double().abs().max() * b.v_scale
    assert ((got[~sees] - clean[~sees]).abs() <= top * (2.0 ** -8 if bf16 else 2.0 ** -17)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16_cache", "e4m3_cache"])
@pytest.mark.parametrize("new,dim", [(3, 128), (100, 64), (100, 128), (100, 256)])
def test_a_part_that_sees_one_key_of_nan(lib, new, dim, e4m3, bf16):
    """The first row's last block of keys is another CTA's part, in which the row sees the first key alone."""
    _nan_key(lib, new, dim, e4m3, bf16, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16_cache", "e4m3_cache"])
@pytest.mark.parametrize("at", [1, 70, 71, 102, 133, 134, 135])
def test_a_key_of_nan_at_any_place_of_a_block(lib, at, e4m3):
    """bf16 outputs of chunks take some of a block's exponentials another way: those have to keep NaN too."""
    for dim in (64, 128, 256):
        _nan_key(lib, 100, dim, e4m3, True, at)
