"""Attention over the paged cache (x_attn_paged) against the plain 64-bit form.

Tolerances, relative to a row's largest |value| that could come out (the largest |v| of its request):
fp32 outputs: a score of size |s| carries 2^-24 |s| per sum step and the exponential 2^-22; scores here
stay below 2^5, so a probability is off by 2^-18 at most, weighted and unweighted alike (twice: above
and below the fraction line). bf16 outputs add a probability's rounding, 2^-9 (fp16 for an e4m3 cache,
2^-12), and the store's, 2^-9 of the value: 2^-8 together with the rest.
"""
import ctypes as C

import numpy as np
import pytest
import torch

import attnref as ref

F32, BF16 = 2.0 ** -17, 2.0 ** -8


def _run(lib, b, q, group, scale, bf16, ldo=None, fill=5.0):
    width = b.heads * group * b.dim
    ldo = ldo or width
    dtype = torch.bfloat16 if bf16 else torch.float32
    out = ref.up(torch.full((b.tokens, ldo), fill, dtype=dtype))
    dq = ref.up(q)
    rc = lib.qwn_x_attn_paged(C.byref(b.cache), C.byref(b.batch), dq.ptr, b.heads * group, scale, out.ptr, ldo, int(bf16))
    assert rc == 0
    lib.tq_sync()
    return ref.down(out, dtype, (b.tokens, ldo))


def _check(lib, b, group, bf16, seed=1, scale=None, ldo=None, big=1.0):
    b.upload()
    scale = b.dim ** -0.5 if scale is None else scale
    q = (torch.randn(b.tokens, b.heads * group, b.dim, generator=b.gen) * big).to(torch.bfloat16)
    got = _run(lib, b, q, group, scale, bf16, ldo)
    assert lib.tq_last_error() == 0
    want = ref.attention(b, q, group, scale)
    n, width = b.start[-1], want.shape[1]
    for r, (new, total) in enumerate(b.lens):
        rows = slice(b.start[r], b.start[r] + new)
        if new:
            top = ref.Batch.rows(b, b.v, r, b.v_scale).abs().max()
            off = (got[rows, :width].double() - want[rows]).abs().max()
            assert off <= top * (BF16 if bf16 else F32), (r, new, total, off / top)
    assert (got[n:] == 5.0).all() and (got[:, width:] == 5.0).all()
    return got


DECODE = [
    # lens, page size, kv heads, group, dim, e4m3
    ([(1, 1)], 16, 1, 1, 64, False),
    ([(1, 15), (1, 16), (1, 17), (1, 64), (1, 65)], 16, 2, 5, 128, False),
    ([(1, 1000), (0, 50), (1, 3), (0, 0), (1, 129)], 48, 4, 6, 256, True),
    ([(1, 700)] * 3, 7, 2, 16, 128, True),
    ([(1, 2500)], 64, 8, 5, 128, False),
    ([(1, 90 + 37 * i) for i in range(20)], 1, 1, 3, 64, True),
    ([(1, 333), (1, 1)], 100, 2, 8, 256, False),
    ([(2, 70), (3, 3), (1, 1), (0, 4)], 16, 2, 4, 128, False),
    ([(4, 600), (2, 31)], 24, 3, 4, 64, False),
    ([(1, 5000)], 32, 1, 1, 128, True),
    ([(1, 200)], 16, 1, 40, 128, False),
]
CHUNKS = [
    ([(128, 128)], 64, 1, 1, 128, False),
    ([(129, 129), (1, 300), (70, 500)], 48, 2, 5, 128, False),
    ([(200, 257), (0, 31), (33, 33)], 16, 2, 3, 256, False),
    ([(65, 400)], 7, 4, 2, 64, True),
    ([(300, 900)], 100, 1, 8, 128, True),
    ([(17, 2000), (16, 16), (1, 1)], 16, 2, 6, 256, True),
    ([(500, 500)], 32, 2, 4, 64, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", DECODE + CHUNKS, ids=[str(i) for i in range(len(DECODE + CHUNKS))])
def test_attention_matches_the_plain_form(lib, case, bf16):
    lens, page, heads, group, dim, e4m3 = case
    _check(lib, ref.Batch(lens, page, heads, dim, e4m3, seed=dim + group, pad=2), group, bf16)


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_never_uses_stale_slots(lib, e4m3, new):
    """NaN in every slot that no request has written, inside its last pages and in unused ones."""
    lens = [(new, 75), (1, 3), (min(new, 17), 130)]
    _check(lib, ref.Batch(lens, 32, 2, 128, e4m3, seed=8, stale=float("nan")), 4, False)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_with_a_wide_output_and_large_scores(lib, dim, new):
    """Rows in a wider matrix, and scores up to some hundreds: one key takes nearly all the weight. A score's
    rounding is 2^-24 of its size then, 2^-15 with 2^9: the bound grows by that."""
    b = ref.Batch([(new, 400), (1, 9)], 16, 2, dim, seed=5).upload()
    q = (torch.randn(b.tokens, 6, dim, generator=b.gen) * 20).to(torch.bfloat16)
    width = 6 * dim
    got = _run(lib, b, q, 3, dim ** -0.5, False, ldo=width + 64)
    want = ref.attention(b, q, 3, dim ** -0.5)
    assert (got[:, width:] == 5.0).all()
    assert (got[:, :width].double() - want).abs().max() <= b.v.abs().max().double() * 2.0 ** -13


@pytest.mark.gpu
def test_attention_negative_and_zero_scale(lib):
    for scale in (0.0, -0.3):
        _check(lib, ref.Batch([(1, 100), (20, 60)], 16, 2, 64, seed=6), 2, False, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16", "e4m3"])
def test_attention_of_queries_of_any_size(lib, e4m3):
    """bf16's range of queries: rows of 2^90 and of 2^-90 among ordinary ones, their scale taken back."""
    b = ref.Batch([(1, 200), (1, 200), (40, 90)], 16, 1, 128, e4m3, seed=12).upload()
    q = torch.randn(b.tokens, 1, 128, generator=b.gen)
    q[0] *= 2.0 ** -90
    q[2] *= 2.0 ** -90
    q = q.to(torch.bfloat16)
    got = _run(lib, b, q, 1, 128 ** -0.5, False)
    want = ref.attention(b, q, 1, 128 ** -0.5)
    assert (got.double() - want).abs().max() <= b.v.double().abs().max() * b.v_scale * F32
    # one query far up: its scores, scaled down by the same power of two
    q = (torch.randn(b.tokens, 1, 128, generator=b.gen) * 2.0 ** 90).to(torch.bfloat16)
    got = _run(lib, b, q, 1, 128 ** -0.5 * 2.0 ** -90, False)
    want = ref.attention(b, q, 1, 128 ** -0.5 * 2.0 ** -90)
    assert (got.double() - want).abs().max() <= b.v.double().abs().max() * b.v_scale * F32


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 200])
def test_attention_gives_the_same_bits_twice_and_in_a_graph(lib, new):
    b = ref.Batch([(new, 3000), (1, 700), (min(new, 9), 50)], 64, 4, 128, seed=2).upload()
    q = torch.randn(b.tokens, 20, 128, generator=b.gen).to(torch.bfloat16)
    one = _run(lib, b, q, 5, 0.1, False)
    two = _run(lib, b, q, 5, 0.1, False)
    assert np.array_equal(ref.bits(one), ref.bits(two))
    # captured, then replayed with other lengths in the same arrays
    dq, out = ref.up(q), ref.up(torch.zeros(b.tokens, 20 * 128))
    assert lib.tq_graph_capture_begin() == 0
    rc = lib.qwn_x_attn_paged(C.byref(b.cache), C.byref(b.batch), dq.ptr, 20, 0.1, out.ptr, 20 * 128, 0)
    graph = lib.tq_graph_capture_end()
    assert rc == 0 and graph
    lib.tq_graph_launch(graph)
    lib.tq_sync()
    assert np.array_equal(ref.bits(ref.down(out, torch.float32, one.shape)), ref.bits(one))
    b.kv_len[:] = [new + 40, 5, 1500]
    b.kv_len[2] = min(b.kv_len[2], 50)
    b.lens = [(n, int(t)) for (n, _), t in zip(b.lens, b.kv_len)]
    lib.tq_h2d(b.dlen.ptr, b.kv_len.ctypes.data, b.kv_len.nbytes)
    lib.tq_graph_launch(graph)
    lib.tq_sync()
    want = ref.attention(b, q, 5, 0.1)
    got = ref.down(out, torch.float32, one.shape)
    lib.tq_graph_destroy(graph)
    assert (got.double() - want).abs().max() <= b.v.abs().max().double() * F32


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 30])
def test_attention_skips_impossible_requests(lib, new):
    lens = [(new, 60), (1, 20), (1, 33)]
    clean = ref.Batch(lens, 16, 2, 64, seed=7)
    q = torch.randn(clean.tokens, 4, 64, generator=clean.gen).to(torch.bfloat16)
    want = ref.attention(clean, q, 2, 0.125)
    for spoil in ("long", "short"):
        b = ref.Batch(lens, 16, 2, 64, seed=7)
        if spoil == "long":
            b.kv_len[1] = b.table.shape[1] * 16 + 1
        if spoil == "short":
            b.kv_len[1] = 0
        b.upload()
        got = _run(lib, b, q, 2, 0.125, False)
        assert lib.tq_last_error() == 10041
        lib.tq_clear_error()
        t = int(clean.start[1])
        assert (got[t] == 5.0).all()
        assert (got[:t].double() - want[:t]).abs().max() <= 8 * F32
    # a page outside the pool: its slots count as zeros, nothing out of range is read
    b = ref.Batch(lens, 16, 2, 64, seed=7)
    page = b.table[1, 0]
    b.table[1, 0] = -5
    b.upload()
    got = _run(lib, b, q, 2, 0.125, False)
    assert lib.tq_last_error() == 10041
    lib.tq_clear_error()
    b.table[1, 0] = page
    b.k[page], b.v[page] = 0.0, 0.0
    assert (got.double() - ref.attention(b, q, 2, 0.125)).abs().max() <= 8 * F32
    if new > 1:                                        # more new tokens than the batch announces
        b = ref.Batch(lens, 16, 2, 64, seed=7)
        b.max_new = 1
        b.upload()
        got = _run(lib, b, q, 2, 0.125, False)
        assert lib.tq_last_error() == 10042
        lib.tq_clear_error()
        assert (got[:new] == 5.0).all()
        assert (got[new:].double() - want[new:]).abs().max() <= 8 * F32


def test_attention_refuses_bad_arguments(pkg):
    lib = pkg.load()
    cache = pkg.KvCache(4096, 4096, 4, 16, 2, 64, 0, 1.0, 1.0)
    batch = pkg.KvBatch(1, 1, 1, 4, 4096, 4096, 4096)
    good = dict(q=4096, heads=4, scale=0.125, out=4096, ldo=256, bf16=0)
    for change, rc in [
        (dict(q=None), -2), (dict(out=None), -2), (dict(heads=0), -2), (dict(heads=3), -3), (dict(ldo=255), -2),
        (dict(ldo=258), -4), (dict(ldo=260, bf16=1), -4), (dict(q=4104), -4), (dict(out=4100), -4),
        (dict(scale=float("nan")), -2), (dict(scale=float("inf")), -2), (dict(bf16=2), -2), (dict(heads=131072), -3),
    ]:
        a = good | change
        assert lib.qwn_x_attn_paged(C.byref(cache), C.byref(batch), a["q"], a["heads"], a["scale"], a["out"], a["ldo"],
                                    a["bf16"]) == rc, change


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("lens", [[(1, 900), (1, 30), (1, 2500), (1, 64)], [(300, 900), (1, 2000), (70, 70)]], ids=["decode", "chunks"])
def test_attention_in_place_of_the_queries(lib, lens, e4m3):
    """bf16 rows over the queries themselves: the bits of the call with an output of its own, tiles cut or not."""
    b = ref.Batch(lens, 16, 2, 128, e4m3, seed=31).upload()
    q = torch.randn(b.tokens, 10, 128, generator=b.gen).to(torch.bfloat16)
    want = _run(lib, b, q, 5, 0.1, True)
    for _ in range(3):
        dq = ref.up(q)
        assert lib.qwn_x_attn_paged(C.byref(b.cache), C.byref(b.batch), dq.ptr, 10, 0.1, dq.ptr, 1280, 1) == 0
        lib.tq_sync()
        assert np.array_equal(ref.bits(ref.down(dq, torch.bfloat16, want.shape)), ref.bits(want))


def test_attention_refuses_an_output_over_its_queries(pkg):
    """4 tokens x 2 heads x 64 values are 1024 bytes of queries."""
    lib = pkg.load()
    cache = pkg.KvCache(4096, 4096, 4, 16, 2, 64, 0, 1.0, 1.0)
    batch = pkg.KvBatch(1, 4, 4, 4, 4096, 4096, 4096)
    q = 1 << 20

    def call(out, ldo, bf16):
        return lib.qwn_x_attn_paged(C.byref(cache), C.byref(batch), q, 2, 0.125, out, ldo, bf16)

    for out, ldo, bf16 in [(q, 128, 0), (q, 136, 1), (q + 16, 128, 1), (q - 1008, 128, 1), (q - 2032, 128, 0), (q + 1008, 128, 1),
                           (q - 2 * (3 * 256 + 128) + 16, 256, 1)]:
        assert call(out, ldo, bf16) == -2, (out - q, ldo, bf16)


def test_attention_refuses_a_scale_that_overflows(pkg):
    """The scale goes by the cache's and into base 2 in fp32."""
    lib = pkg.load()
    batch = pkg.KvBatch(1, 1, 1, 4, 4096, 4096, 4096)
    for k_scale, e4m3, scale in [(2.0 ** 100, 1, 2.0 ** 100), (1.0, 0, 3e38), (1.0, 0, -3e38)]:
        cache = pkg.KvCache(4096, 4096, 4, 16, 2, 64, e4m3, k_scale, 1.0)
        assert lib.qwn_x_attn_paged(C.byref(cache), C.byref(batch), 8192, 2, scale, 4096, 128, 0) == -2, (k_scale, scale)


def _many(count, longest, seed):
    """Requests of one token, one in five without any, lengths over the whole range."""
    g = np.random.default_rng(seed)
    return [(int(i % 5 != 3), int(g.integers(1, longest))) for i in range(count)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    # more requests than the decode kernel has threads, across one and several blocks of them
    (_many(129, 60, 1), 16, 2, 4, 64, False),
    (_many(300, 200, 2), 16, 1, 8, 128, True),
    (_many(700, 40, 3), 7, 2, 1, 256, False),
    ([(0, 5)] * 256 + [(1, 90)] + [(0, 0)] * 200 + [(1, 7)], 16, 2, 2, 64, False),
    # and than the kernel for chunks has
    (_many(460, 60, 4) + [(150, 300)] + _many(50, 90, 5), 16, 2, 2, 128, False),
    (_many(500, 40, 6) + [(40, 40)], 20, 1, 6, 64, False),
    ([(30, 45)] + _many(470, 40, 7) + [(90, 333)], 16, 1, 2, 256, True),
    # a request of more row tiles than that has threads
    ([(3, 9), (700, 700), (1, 40)], 64, 1, 64, 64, False),
], ids=[str(i) for i in range(8)])
def test_attention_of_more_requests_and_tiles_than_threads(lib, case):
    lens, page, heads, group, dim, e4m3 = case
    for bf16 in (False, True):
        _check(lib, ref.Batch(lens, page, heads, dim, e4m3, seed=len(lens)), group, bf16)


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16", "e4m3"])
def test_attention_of_a_mixed_step_in_two_calls(lib, pkg, e4m3):
    """Single tokens, then chunks: a record of each sort's requests over the same arrays. Rows of the other sort stay."""
    lens = [(1, 700), (1, 3), (0, 90), (1, 1200), (60, 300), (0, 0), (150, 150)]
    b = ref.Batch(lens, 16, 2, 128, e4m3, seed=77, pad=3).upload()
    q = torch.randn(b.tokens, 10, 128, generator=b.gen).to(torch.bfloat16)
    want = ref.attention(b, q, 5, 0.1)
    dq, out = ref.up(q), ref.up(torch.full((b.tokens, 1280), 5.0))
    cut, n = 4, len(lens)
    for r0, r1, most in ((0, cut, 1), (cut, n, 150)):
        part = pkg.KvBatch(r1 - r0, b.tokens, most, b.table.shape[1], b.dstart.ptr + 4 * r0, b.dlen.ptr + 4 * r0,
                           b.dtable.ptr + 4 * r0 * b.table.shape[1])
        assert lib.qwn_x_attn_paged(C.byref(b.cache), C.byref(part), dq.ptr, 10, 0.1, out.ptr, 1280, 0) == 0
        lib.tq_sync()
        assert lib.tq_last_error() == 0
        got = ref.down(out, torch.float32, (b.tokens, 1280))
        done = slice(0, b.start[r1])
        assert (got[done].double() - want[done]).abs().max() <= b.v.double().abs().max() * b.v_scale * F32
        assert (got[b.start[r1]:] == 5.0).all()
