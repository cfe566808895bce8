"""Low-rank adapters beside a projection (x_lora_add) against the plain 64-bit form.

Tolerance: products are exact (bf16 weights, x and h in all their 24 bits), sums are fp32 with at most
2^-24 relative to the running sum's size per step. A value of h sums K products in K/16 steps over a few
accumulators, a value of y rank more and the base: against the sum of the absolute products that bounds a
running sum, (K / 16 + rank + 8) 2^-24.
"""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import attnref as ref


def _make(pkg, count, adapters, rank, Ms, K, T, ids, ranks=True, scales=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    c = {"x": torch.randn(T, K, generator=g), "ids": torch.tensor(ids, dtype=torch.int32), "w": []}
    c["x"][:, ::97] *= 20.0
    for i in range(count):
        w = {"a": (torch.randn(adapters, rank, K, generator=g) * K ** -0.5).to(torch.bfloat16),
             "b": (torch.randn(adapters, Ms[i], rank, generator=g) * 0.1).to(torch.bfloat16),
             "rank": torch.randint(0, rank + 1, (adapters,), generator=g, dtype=torch.int32) if ranks else None,
             "scale": torch.rand(adapters, generator=g) + 0.5 if scales else None,
             "base": torch.randn(T, Ms[i], generator=g)}
        if ranks:                       # what lies beyond an adapter's rank must not be used
            w["rank"][0] = rank
            for j in range(adapters):
                w["a"][j, int(w["rank"][j]):] = float("nan")
                w["b"][j, :, int(w["rank"][j]):] = float("nan")
        w["dev"] = [ref.up(w["a"]), ref.up(w["b"]), ref.up(w["rank"]) if ranks else None,
                    ref.up(w["scale"]) if scales else None]
        p = [d.ptr if d else None for d in w["dev"]]
        w["rec"] = pkg.Lora(adapters, rank, Ms[i], K, *p)
        c["w"].append(w)
    return c


def _run(lib, pkg, c, base="own"):
    T = c["x"].shape[0]
    x, ids = ref.up(c["x"]), ref.up(c["ids"])
    if base == "inplace":
        ys = [ref.up(w["base"]) for w in c["w"]]
        bases = ys
    else:
        ys = [ref.up(torch.full_like(w["base"], 3.0)) for w in c["w"]]
        bases = [ref.up(w["base"]) for w in c["w"]] if base == "own" else None
    n = len(ys)
    rc = lib.qwn_x_lora_add(pkg.lora_array([w["rec"] for w in c["w"]]), ref.ptrs(bases) if bases else None, ref.ptrs(ys),
                            n, x.ptr, ids.ptr, T)
    assert rc == 0
    lib.tq_sync()
    return [ref.down(y, torch.float32, w["base"].shape) for y, w in zip(ys, c["w"])]


def _check(got, c, base=True):
    K = c["x"].shape[1]
    for y, w in zip(got, c["w"]):
        a, b = torch.nan_to_num(w["a"].float()), torch.nan_to_num(w["b"].float())
        bs = w["base"] if base else None
        want = ref.lora(c["x"], c["ids"], a, b, w["rank"], w["scale"], bs)
        size = ref.lora(c["x"].abs(), c["ids"], a.abs(), b.abs(), w["rank"], w["scale"], bs.abs() if base else None)
        steps = K / 16 + a.shape[1] + 8
        off = (y.double() - want).abs()
        assert (off <= size * steps * 2.0 ** -24 + 1e-30).all(), (off / size.clamp(min=1e-30)).max() * 2.0 ** 24


CASES = [
    # projections' rows, adapters, rank, K, T
    ([16], 1, 8, 32, 1),
    ([1024], 4, 16, 5120, 1),
    ([48, 272], 3, 24, 96, 5),
    ([512, 64, 64], 7, 64, 1024, 33),
    ([256], 40, 32, 512, 64),
    ([144], 2, 256, 256, 17),
    ([320, 320], 5, 72, 2080, 130),
    ([1040], 3, 40, 640, 700),
    ([64, 32, 16, 48], 300, 8, 64, 200),
    ([2560, 1296], 3, 72, 64, 3000),
    ([1920], 30, 64, 96, 4500),
    ([96], 3, 24, 9248, 40),
    ([64, 48], 2, 32, 1120, 333),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("base", ["own", "inplace", "none"])
def test_lora_matches_the_plain_form(lib, pkg, case, base):
    Ms, n, rank, K, T = case
    rng = np.random.default_rng(T + K)
    ids = rng.integers(-1, n, T)
    c = _make(pkg, len(Ms), n, rank, Ms, K, T, ids, seed=T)
    _check(_run(lib, pkg, c, base), c, base != "none")
    assert lib.tq_last_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("ids", [[-1] * 40, [2] * 40, list(range(4)) * 10, [-1] * 39 + [0], [0] + [-7] * 39])
def test_lora_orders_of_tokens(lib, pkg, ids):
    """No adapter at all, one for all tokens, one after another, a single token with one; without rank and scale arrays."""
    c = _make(pkg, 2, 4, 16, [96, 80], 160, 40, ids, ranks=False, scales=False, seed=3)
    got = _run(lib, pkg, c)
    _check(got, c)
    for y, w in zip(got, c["w"]):       # without an adapter the base's bits come out
        none = c["ids"] < 0
        assert torch.equal(y[none], w["base"][none])


@pytest.mark.gpu
def test_lora_in_place_without_any_adapter(lib, pkg):
    """Nothing to do for any row: all of them keep their bits, and the next call works."""
    c = _make(pkg, 2, 4, 16, [96, 80], 160, 70, [-1] * 70, seed=4)
    for y, w in zip(_run(lib, pkg, c, "inplace"), c["w"]):
        assert torch.equal(y, w["base"])
    c = _make(pkg, 2, 4, 16, [96, 80], 160, 70, [t % 5 - 1 for t in range(70)], seed=5)
    _check(_run(lib, pkg, c, "inplace"), c)
    assert lib.tq_last_error() == 0


@pytest.mark.gpu
def test_lora_rows_do_not_depend_on_their_company(lib, pkg):
    """Values that are not finite stay in their own token's row, and a token's bits do not depend on who
    shares its tile."""
    T = 24
    c = _make(pkg, 1, 2, 16, [64], 128, T, [0] * T, ranks=False, seed=5)
    clean = _run(lib, pkg, c)[0]
    c["x"][3, 5], c["x"][9, 0] = float("nan"), float("inf")
    got = _run(lib, pkg, c)[0]
    keep = [t for t in range(T) if t not in (3, 9)]
    assert torch.equal(got[keep], clean[keep])
    assert not torch.isfinite(got[[3, 9]]).any()
    c["ids"][:12] = -1
    c["x"][3, 5], c["x"][9, 0] = 0.0, 0.0
    assert torch.equal(_run(lib, pkg, c)[0][12:], clean[12:])


@pytest.mark.gpu
def test_lora_largest_finite_inputs(lib, pkg):
    """x near fp32's largest value: the terms it enters the tensor core with do not overflow."""
    c = _make(pkg, 1, 1, 8, [16], 32, 1, [0], ranks=False, scales=False, seed=6)
    c["x"].zero_()
    c["x"][0, 3] = 3.4028234663852886e38
    c["w"][0]["dev"][0] = ref.up((c["w"][0]["a"].float() * 2.0 ** -40).to(torch.bfloat16))
    c["w"][0]["a"] = (c["w"][0]["a"].float() * 2.0 ** -40).to(torch.bfloat16)
    c["w"][0]["rec"].d_a = c["w"][0]["dev"][0].ptr
    _check(_run(lib, pkg, c), c)


@pytest.mark.gpu
def test_lora_numbers_out_of_range_count_as_none(lib, pkg):
    c = _make(pkg, 1, 3, 16, [64], 64, 6, [0, 3, 1, 99, 2, -1], seed=7, ranks=False)
    got = _run(lib, pkg, c)[0]
    assert lib.tq_last_error() == 10043
    lib.tq_clear_error()
    assert torch.equal(got[[1, 3, 5]], c["w"][0]["base"][[1, 3, 5]])
    c["ids"][[1, 3]] = -1
    _check([got], c)
    c["w"][0]["rank"] = torch.tensor([16, 17, -1], dtype=torch.int32)
    c["w"][0]["dev"][2] = ref.up(c["w"][0]["rank"])
    c["w"][0]["rec"].d_rank = c["w"][0]["dev"][2].ptr
    got = _run(lib, pkg, c)[0]
    assert lib.tq_last_error() == 10043
    lib.tq_clear_error()
    c["w"][0]["rank"] = torch.tensor([16, 0, 0], dtype=torch.int32)
    _check([got], c)


@pytest.mark.gpu
def test_lora_in_a_graph(lib, pkg):
    c = _make(pkg, 2, 3, 16, [64, 48], 96, 9, [0, 1, 2, -1, 0, 0, 1, 2, 2], seed=8)
    first = _run(lib, pkg, c)                       # the scratch is there now
    x, ids = ref.up(c["x"]), ref.up(c["ids"])
    ys, bases = ([ref.up(w["base"]) for w in c["w"]] for _ in range(2))
    assert lib.tq_graph_capture_begin() == 0
    rc = lib.qwn_x_lora_add(pkg.lora_array([w["rec"] for w in c["w"]]), ref.ptrs(bases), ref.ptrs(ys), 2, x.ptr, ids.ptr, 9)
    graph = lib.tq_graph_capture_end()
    assert rc == 0 and graph
    lib.tq_graph_launch(graph)
    c["ids"] = torch.tensor([1, 1, -1, 0, 2, 2, 0, 0, 1], dtype=torch.int32)
    lib.tq_sync()
    for y, f in zip(ys, first):
        assert np.array_equal(ref.bits(ref.down(y, torch.float32, f.shape)), ref.bits(f))
    v = c["ids"].numpy()
    lib.tq_h2d(ids.ptr, v.ctypes.data, v.nbytes)
    lib.tq_graph_launch(graph)
    lib.tq_sync()
    lib.tq_graph_destroy(graph)
    _check([ref.down(y, torch.float32, f.shape) for y, f in zip(ys, first)], c)


GROWTH = """
import ctypes as C, importlib, sys
sys.path[:0] = [{root!r}, {root!r} + "/tests"]
import torch
import attnref as ref
from test_lora import _make, _run, _check
pkg = importlib.import_module("knivesysl-xe_b200")
lib = pkg.load()
assert lib.tq_set_device(0) == 0
c = _make(pkg, 1, 2, 8, [64], 64, 3, [0, 1, 0], seed=1)
_run(lib, pkg, c)
x, ids, base, y = ref.up(c["x"]), ref.up(c["ids"]), ref.up(c["w"][0]["base"]), ref.up(c["w"][0]["base"])
assert lib.tq_graph_capture_begin() == 0
assert lib.qwn_x_lora_add(pkg.lora_array([c["w"][0]["rec"]]), ref.ptrs([base]), ref.ptrs([y]), 1, x.ptr, ids.ptr, 3) == 0
graph = lib.tq_graph_capture_end()
keep = []
for T in (70, 600, 3000):                  # each wants more scratch than the last
    d = _make(pkg, 2, 2, 128, [64, 64], 128, T, [t % 2 for t in range(T)], seed=T)
    _check(_run(lib, pkg, d), d)
    other = pkg.DevBuf(1 << 16)            # would take the place of what was freed
    lib.tq_dev_fill(other.ptr, 0x5a, other.nbytes)
    keep.append(other)
lib.tq_graph_launch(graph)
lib.tq_sync()
lib.tq_graph_destroy(graph)
_check([ref.down(y, torch.float32, (3, 64))], c)
for other in keep:
    assert (other.to_numpy("uint8", 1 << 16) == 0x5a).all()
assert lib.tq_last_error() == 0
print("ok")
"""


@pytest.mark.gpu
def test_a_captured_call_outlives_larger_ones(lib):
    """The scratch that a graph was captured with is not given back when a larger call makes a new one."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", GROWTH.format(root=root)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.splitlines() == ["ok"], out.stderr


FIRST_CALL = """
import ctypes as C, importlib, sys
sys.path.insert(0, {root!r})
pkg = importlib.import_module("knivesysl-xe_b200")
lib = pkg.load()
assert lib.tq_set_device(0) == 0
buf = pkg.DevBuf(1 << 20)
lib.tq_dev_fill(buf.ptr, 0, buf.nbytes)
lib.tq_sync()
p = buf.ptr
cache = pkg.KvCache(p, p + 65536, 4, 16, 2, 64, 0, 1.0, 1.0)
batch = pkg.KvBatch(1, 1, 1, 4, p, p, p)
one = (C.c_void_p * 1)(p + 262144)
ws = pkg.lora_array([pkg.Lora(1, 8, 16, 32, p, p, None, None)])
calls = dict(
    append=lambda: lib.qwn_x_kv_append(C.byref(cache), C.byref(batch), None, None, 0, 0, None, p, 128, p, 128),
    attend=lambda: lib.qwn_x_attn_paged(C.byref(cache), C.byref(batch), p, 2, 0.125, p + 131072, 128, 0),
    lora=lambda: lib.qwn_x_lora_add(ws, None, one, 1, p, p, 1))
assert lib.tq_graph_capture_begin() == 0
got = calls[{call!r}]()
graph = lib.tq_graph_capture_end()
print("first", got, lib.tq_last_error())
print("then", calls[{call!r}]())
lib.tq_sync()
print("end", lib.tq_last_error())
"""


@pytest.mark.gpu
@pytest.mark.parametrize("call", ["append", "attend", "lora"])
def test_a_first_call_inside_a_capture_is_refused(lib, call):
    """Memory cannot be allocated while the stream is captured: -40, no abort, and the next call works. (A batch of
    zeros: one request without tokens; all-zero adapters.)"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", FIRST_CALL.format(root=root, call=call)], capture_output=True, text=True,
                         timeout=120)
    assert out.returncode == 0, out.stderr
    assert out.stdout.splitlines() == ["first -40 0", "then 0", "end 0"], out.stdout


def test_lora_refuses_bad_arguments(pkg):
    lib = pkg.load()
    rec = dict(count=2, rank=16, M=64, K=64, d_a=4096, d_b=4096, d_rank=None, d_scale=None)
    one = (C.c_void_p * 1)(4096)
    for change, rc in [
        (dict(count=0), -1), (dict(rank=0), -1), (dict(M=0), -1), (dict(K=0), -1), (dict(d_a=None), -1), (dict(d_b=None), -1),
        (dict(K=48), -3), (dict(M=24), -3), (dict(rank=12), -3), (dict(rank=264), -3), (dict(count=2049), -3),
        (dict(d_a=4104), -4), (dict(d_b=4098), -4),
    ]:
        ws = pkg.lora_array([pkg.Lora(**(rec | change))])
        assert lib.qwn_x_lora_add(ws, one, one, 1, 4096, 4096, 4) == rc, change
    ws = pkg.lora_array([pkg.Lora(**rec)])
    assert lib.qwn_x_lora_add(None, one, one, 1, 4096, 4096, 4) == -2
    assert lib.qwn_x_lora_add(ws, one, None, 1, 4096, 4096, 4) == -2
    assert lib.qwn_x_lora_add(ws, one, one, 0, 4096, 4096, 4) == -2
    assert lib.qwn_x_lora_add(ws, one, one, 5, 4096, 4096, 4) == -2
    assert lib.qwn_x_lora_add(ws, one, one, 1, None, 4096, 4) == -2
    assert lib.qwn_x_lora_add(ws, one, one, 1, 4096, None, 4) == -2
    assert lib.qwn_x_lora_add(ws, one, one, 1, 4096, 4096, -1) == -2
    assert lib.qwn_x_lora_add(ws, one, (C.c_void_p * 1)(None), 1, 4096, 4096, 4) == -2
    assert lib.qwn_x_lora_add(ws, one, one, 1, 4100, 4096, 4) == -4
    assert lib.qwn_x_lora_add(ws, one, (C.c_void_p * 1)(4104), 1, 4096, 4096, 4) == -4
    two = pkg.lora_array([pkg.Lora(**rec), pkg.Lora(**(rec | dict(K=96)))])
    pair = (C.c_void_p * 2)(4096, 4096)
    assert lib.qwn_x_lora_add(two, pair, pair, 2, 4096, 4096, 4) == -2
    assert lib.qwn_x_lora_add(ws, one, one, 1, 4096, 4096, 0) == 0
    # one output twice, an output that is another projection's base, one that is x, more rows of B than 32 bits count
    same = pkg.lora_array([pkg.Lora(**rec)] * 2)
    ys = lambda *p: (C.c_void_p * 2)(*p)
    assert lib.qwn_x_lora_add(same, None, ys(8192, 8192), 2, 4096, 4096, 4) == -2
    assert lib.qwn_x_lora_add(same, ys(12288, 8192), ys(8192, 12288), 2, 4096, 4096, 4) == -2
    assert lib.qwn_x_lora_add(ws, None, one, 1, 4096, 4096, 4) == -2
    wide = pkg.lora_array([pkg.Lora(**(rec | dict(count=2048, M=1 << 20)))])
    assert lib.qwn_x_lora_add(wide, None, (C.c_void_p * 1)(8192), 1, 4096, 4096, 4) == -3


def test_lora_refuses_outputs_that_overlap(pkg):
    """In part, as much as by the same address: T = 4 rows of 64 values are 1024 bytes."""
    lib = pkg.load()
    rec = pkg.Lora(2, 16, 64, 64, 4096, 4096, None, None)
    two = pkg.lora_array([rec, rec])
    x = 1 << 20
    ptrs = lambda *p: (C.c_void_p * len(p))(*p)  # noqa: E731

    def call(ys, bases=None, n=1):
        return lib.qwn_x_lora_add(two, ptrs(*bases) if bases else None, ptrs(*ys), n, x, 4096, 4)

    for y in (x - 1008, x, x + 16, x + 1008):
        assert call([y]) == -2, y
    for base in (8192 - 1008, 8192 + 256):                       # rows of the base that other rows' results overwrite
        assert call([8192], [base]) == -2, base
    for y in (8192 - 1008, 8192 + 512):
        assert call([8192, y], n=2) == -2, y
        assert call([8192, 65536], [None, y], n=2) == -2, y
