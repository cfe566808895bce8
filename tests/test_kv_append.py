"""Keys and values into the paged cache (x_kv_append) against the plain 64-bit form.

Tolerances: a stored value is rounded once, by half a step at most (bf16 2^-9 of the value's power of
two, 2^-8 of the value itself; e4m3 2^-4), after an fp32 computation. That one's error is 2^-24 per
operation: the angle in 64 bits leaves 2^-24 of pi, the norm's sum and root some 2^-21; together below
2^-19 of the pair's or row's size, which can also move a value across a rounding border.
"""
import ctypes as C

import numpy as np
import pytest
import torch

import attnref as ref

EPS = 2.0 ** -19


def _call(lib, b, qkv, q_heads, rope, pad_q=True):
    D, H, Hk = b.dim, q_heads, b.heads
    width = qkv.shape[1]
    x = ref.up(qkv)
    guard = torch.full((b.tokens, max(1, H), D), 7.0, dtype=torch.bfloat16)
    q_out = ref.up(guard)
    rc = lib.qwn_x_kv_append(C.byref(b.cache), C.byref(b.batch), C.byref(rope) if rope else None,
                             x.ptr if H else None, width, H, q_out.ptr if H else None, x.ptr + 4 * H * D, width,
                             x.ptr + 4 * (H + Hk) * D, width)
    assert rc == 0
    lib.tq_sync()
    shape = (b.pages, Hk, b.page_size, D)
    return (ref.down(q_out, torch.bfloat16, guard.shape), ref.down(b.dk, b.dtype, shape), ref.down(b.dv, b.dtype, shape))


def _near(got, want, half_step, size):
    """Within half a step of the rounding, and the computation's own error in units of the row's size."""
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    off = (got - want).abs() - want.abs() * half_step
    assert (torch.nan_to_num(off) <= size * EPS).all(), (off - size * EPS).max()


CASES = [
    # lens, page size, q heads, kv heads, dim, rot, interleaved, norm, e4m3
    ([(1, 1)], 16, 1, 1, 64, 64, False, False, False),
    ([(1, 1), (1, 17), (0, 9), (1, 33)], 16, 10, 2, 128, 128, False, True, False),
    ([(5, 5), (0, 0), (3, 40), (1, 7)], 7, 6, 2, 128, 48, True, True, True),
    ([(33, 70), (2, 2)], 1, 4, 4, 256, 64, False, False, True),
    ([(70, 300)], 100, 24, 4, 256, 256, True, False, False),
    ([(9, 20), (1, 1000)], 64, 32, 4, 64, 32, False, True, True),
    ([(640, 1000)], 48, 8, 8, 64, 16, False, True, False),
    ([(1, 3)] * 70, 8, 5, 1, 128, 0, False, True, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_append_matches_the_plain_form(lib, pkg, case):
    lens, page, H, Hk, D, rot, inter, norm, e4m3 = case
    b = ref.Batch(lens, page, Hk, D, e4m3, seed=len(lens) + D, pad=3).upload()
    qkv = torch.randn(b.tokens, (H + 2 * Hk) * D, generator=b.gen)
    inv = 1e4 ** (-torch.arange(0, max(rot, 2), 2).double() / max(rot, 2))
    inv = inv.float()
    wq, wk = ((torch.randn(D, generator=b.gen) * 0.1).to(torch.bfloat16) if norm else None for _ in range(2))
    keep = [ref.up(inv)] + ([ref.up(wq), ref.up(wk)] if norm else [])
    rope = pkg.Rope(keep[0].ptr, rot, int(inter), keep[1].ptr if norm else None, keep[2].ptr if norm else None, 1e-6)
    q, k, v = _call(lib, b, qkv, H, rope)
    assert lib.tq_last_error() == 0
    wq64, wk64, wv64 = ref.append(b, qkv, H, inv, rot, inter, wq, wk)
    n = b.start[-1]
    assert (q[n:] == 7.0).all()                       # padding rows are left alone
    _near(q[:n], wq64[:n], 2.0 ** -8, 8.0)
    step = 2.0 ** -4 if e4m3 else 2.0 ** -8
    # below e4m3's normal range a step is 2^-9 of a stored unit
    floor = 2.0 ** -10 / EPS if e4m3 else 8.0
    _near(k, wk64, step, max(8.0 / b.k_scale, floor))
    _near(v, wv64, step, max(1e-30, floor if e4m3 else 1e-30))
    # what no new token owns keeps its bits
    own = torch.zeros(b.pages, page, dtype=torch.bool)
    for r, (new, total) in enumerate(lens):
        p = np.arange(total - new, total)
        own[b.table[r, p // page], p % page] = True
    rest = ~own[:, None, :].expand(-1, Hk, -1)
    for got, was in ((k, b.k), (v, b.v)):
        assert np.array_equal(ref.bits(got.float()[rest]), ref.bits(was.float()[rest]))


@pytest.mark.gpu
def test_append_far_positions_keep_their_angles(lib, pkg):
    """At position two million the angle is a product of 64 bits: an fp32 one would be off by 0.1."""
    D, pos = 128, 2_000_000
    b = ref.Batch([(1, 5)], 8, 1, D, seed=3)
    b.page_size, b.table = 8, np.full((1, (pos + 8) // 8), 0, np.int32)
    b.kv_len, b.lens = np.array([pos + 1], np.int32), [(1, pos + 1)]
    b.upload()
    qkv = torch.randn(1, 3 * D, generator=b.gen)
    inv = (1e6 ** (-torch.arange(0, D, 2).double() / D)).float()
    d = ref.up(inv)
    q, k, v = _call(lib, b, qkv, 1, pkg.Rope(d.ptr, D, 0, None, None, 0.0))
    want, _, _ = ref.append(b, qkv, 1, inv, D, False)
    _near(q, want, 2.0 ** -8, 8.0)


@pytest.mark.gpu
def test_append_without_rope_saturates_e4m3_and_takes_keys_alone(lib):
    b = ref.Batch([(2, 3)], 4, 1, 64, True, seed=9, scales=(1.0, 1.0)).upload()
    qkv = torch.randn(2, 128, generator=b.gen)
    qkv[0, :4] = torch.tensor([1e6, -1e6, 448.0, 464.0])
    _, k, v = _call(lib, b, qkv, 0, None)
    at = b.table[0, 0], 0, 1
    assert k[at].float()[:4].tolist() == [448.0, -448.0, 448.0, 448.0]
    assert np.array_equal(ref.bits(k[at][4:]), ref.bits(qkv[0, 4:64].to(torch.float8_e4m3fn)))
    assert np.array_equal(ref.bits(v[at]), ref.bits(qkv[0, 64:].to(torch.float8_e4m3fn)))


@pytest.mark.gpu
def test_append_skips_what_the_arrays_cannot_mean(lib):
    """A page outside the pool, a range that leaves the matrix: nothing of it is stored, the rest is."""
    for spoil in ("page", "range", "short", "most"):
        b = ref.Batch([(2, 6), (1, 4)], 4, 2, 64, seed=4)
        if spoil == "page":
            b.table[0, 1] = b.pages
        if spoil == "range":
            b.start[:] = [0, 2, 99]
        if spoil == "short":
            b.kv_len[0] = 1
        if spoil == "most":
            b.max_new = 1
        b.upload()
        qkv = torch.randn(b.tokens, 6 * 64, generator=b.gen)
        _, k, _ = _call(lib, b, qkv, 2, None)
        assert lib.tq_last_error() == (10042 if spoil == "most" else 10041)
        lib.tq_clear_error()
        skipped, stored = (1, 0) if spoil == "range" else (0, 1)
        good = ref.Batch([(2, 6), (1, 4)], 4, 2, 64, seed=4)
        new = {0: [(good.table[0, 1], 0), (good.table[0, 1], 1)], 1: [(good.table[1, 0], 3)]}
        for page, slot in new[skipped]:
            assert torch.equal(k[page, :, slot].float(), b.k[page, :, slot].float())
        t = int(good.start[stored])
        for i, (page, slot) in enumerate(new[stored]):
            assert torch.equal(k[page, :, slot], qkv[t + i, 128:256].view(2, 64).to(torch.bfloat16))


def _fake(pkg, **change):
    f = {"cache": dict(d_k=4096, d_v=4096, pages=4, page_size=16, heads=2, dim=64, e4m3=0, k_scale=1.0, v_scale=1.0),
         "batch": dict(count=1, tokens=1, max_new=1, max_pages=4, d_start=4096, d_kv_len=4096, d_pages=4096)}
    for key, value in change.items():
        part, name = key.split("_", 1)
        f[part][name] = value
    return pkg.KvCache(**f["cache"]), pkg.KvBatch(**f["batch"])


BAD_RECORDS = [
    (dict(cache_d_k=None), -1), (dict(cache_pages=0), -1), (dict(cache_page_size=0), -1), (dict(cache_heads=0), -1),
    (dict(cache_e4m3=2), -1), (dict(cache_e4m3=1, cache_k_scale=0.0), -1), (dict(cache_dim=96), -3),
    (dict(cache_d_v=4104), -4), (dict(batch_count=-1), -2), (dict(batch_tokens=-1), -2), (dict(batch_max_new=-1), -2),
    (dict(batch_d_start=None), -2), (dict(batch_d_pages=None), -2), (dict(batch_max_pages=0), -2),
    (dict(batch_max_pages=2 ** 28), -3),
    (dict(cache_e4m3=1, cache_v_scale=float("inf")), -1), (dict(cache_e4m3=1, cache_v_scale=float("nan")), -1),
]


@pytest.mark.parametrize("change,rc", BAD_RECORDS, ids=[str(i) for i in range(len(BAD_RECORDS))])
def test_append_and_attention_refuse_bad_records(pkg, change, rc):
    lib = pkg.load()
    cache, batch = _fake(pkg, **change)
    assert lib.qwn_x_kv_append(C.byref(cache), C.byref(batch), None, None, 0, 0, None, 4096, 128, 4096, 128) == rc
    assert lib.qwn_x_attn_paged(C.byref(cache), C.byref(batch), 4096, 2, 0.125, 4096, 128, 0) == rc


def test_append_refuses_bad_arguments(pkg):
    lib = pkg.load()
    cache, batch = _fake(pkg)
    c, b = C.byref(cache), C.byref(batch)
    R = pkg.Rope
    good = dict(rope=None, q=4096, ldq=128, heads=2, out=4096, k=4096, ldk=128, v=4096, ldv=128)
    for change, rc in [
        (dict(q=None), -2), (dict(out=None), -2), (dict(heads=0), -2), (dict(heads=-1), -2), (dict(ldq=127), -2),
        (dict(k=None), -2), (dict(v=None), -2), (dict(ldk=64), -2), (dict(ldv=64), -2), (dict(q=4100), -4),
        (dict(out=4104), -4), (dict(ldk=130), -4), (dict(v=4100), -4), (dict(heads=70000, ldq=1 << 30), -3),
        (dict(rope=R(4096, 24, 0, None, None, 0.0)), -3), (dict(rope=R(4096, 80, 0, None, None, 0.0)), -3),
        (dict(rope=R(None, 64, 0, None, None, 0.0)), -1), (dict(rope=R(4096, 64, 0, 4096, None, -1.0)), -1),
    ]:
        a = good | change
        got = lib.qwn_x_kv_append(c, b, C.byref(a["rope"]) if a["rope"] else None, a["q"], a["ldq"], a["heads"],
                                  a["out"], a["k"], a["ldk"], a["v"], a["ldv"])
        assert got == rc, change
    # nothing to do is no error, and touches no GPU
    cache, batch = _fake(pkg, batch_tokens=0)
    assert lib.qwn_x_kv_append(C.byref(cache), C.byref(batch), None, None, 0, 0, None, 4096, 128, 4096, 128) == 0
    assert lib.qwn_x_attn_paged(C.byref(cache), C.byref(batch), 4096, 2, 0.125, 4096, 128, 0) == 0


def test_append_refuses_queries_out_over_its_inputs(pkg):
    """One token, 2 heads of 64: 256 bytes of queries out, 512 of q rows and 512 of k and of v rows."""
    lib = pkg.load()
    cache, batch = _fake(pkg)
    q, k, v = 1 << 20, 2 << 20, 3 << 20
    for out in (q, q + 496, q - 240, k, k + 256, v - 240, v + 496):
        assert lib.qwn_x_kv_append(C.byref(cache), C.byref(batch), None, q, 128, 2, out, k, 128, v, 128) == -2, out
