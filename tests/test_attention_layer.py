"""An attention layer of a served step, as its operators are used together: projections with adapters, append,
attention, output projection with an adapter. Each stage is compared with the 64-bit form of the stage before it as
the GPU left it; the whole is captured into a graph and replayed."""
import ctypes as C

import numpy as np
import pytest
import torch

import attnref as ref


class Layer:
    def __init__(self, pkg, wl, lens, e4m3, seed):
        g = self.gen = torch.Generator().manual_seed(seed)
        self.pkg, self.hidden, self.heads, self.kv, self.dim = pkg, 320, 4, 2, 64
        self.b = ref.Batch(lens, 16, self.kv, self.dim, e4m3, seed=seed)
        self.T = self.b.tokens
        assert self.T % 8 == 0
        self.x = torch.randn(self.T, self.hidden, generator=g)
        self.rows = [self.heads * 64, self.kv * 64, self.kv * 64]
        self.w = [self._weight(wl, m, self.hidden, i) for i, m in enumerate(self.rows)]
        self.wo = self._weight(wl, self.hidden, self.heads * 64, 9)
        self.ids = torch.randint(-1, 3, (self.T,), generator=g, dtype=torch.int32)
        self.lora = [self._lora(m, self.hidden) for m in self.rows]
        self.lora_o = self._lora(self.hidden, self.heads * 64)
        self.inv = (1e4 ** (-torch.arange(0, 32, 2).double() / 32)).float()
        self.qn, self.kn = ((torch.randn(64, generator=g) * 0.1).to(torch.bfloat16) for _ in range(2))

    def _weight(self, wl, M, K, seed):
        codes, scales = wl.make_weight_w4(M, K, seed=seed + 40, group=32)
        return self.pkg.PackedWeight(codes, scales, M, K)

    def _lora(self, M, K):
        a = (torch.randn(3, 16, K, generator=self.gen) * K ** -0.5).to(torch.bfloat16)
        b = (torch.randn(3, M, 16, generator=self.gen) * 0.1).to(torch.bfloat16)
        dev = [ref.up(a), ref.up(b)]
        return {"a": a, "b": b, "dev": dev, "rec": self.pkg.Lora(3, 16, M, K, dev[0].ptr, dev[1].ptr, None, None)}

    def upload(self):
        p, T = self.pkg, self.T
        self.b.upload()
        f = lambda *s: p.DevBuf(4 * int(np.prod(s)))  # noqa: E731
        self.dx, self.dids, self.dinv, self.dqn, self.dkn = (ref.up(t) for t in (self.x, self.ids, self.inv, self.qn, self.kn))
        self.qkv, self.q, self.o, self.y = [f(T, m) for m in self.rows], p.DevBuf(2 * T * self.rows[0]), f(T, self.rows[0]), \
            f(T, self.hidden)
        n = max(self.hidden, self.rows[0]) // 32 * T
        self.aq, self.as_, self.asum = p.DevBuf(n * 32), f(n), f(n)
        self.rope = p.Rope(self.dinv.ptr, 32, 0, self.dqn.ptr, self.dkn.ptr, 1e-6)

    def project(self, lib):
        lib.qwn_x_quantize_act_chunk(self.dx.ptr, self.hidden, self.T, self.aq.ptr, self.as_.ptr, self.asum.ptr)
        assert lib.qwn_x_gemm_w4a8_fanout(self.pkg.weight_array(self.w), ref.ptrs(self.qkv), 3, self.aq.ptr, self.as_.ptr,
                                          self.asum.ptr, self.T, None, 0) == 0

    def adapt(self, lib):
        ys = ref.ptrs(self.qkv)
        assert lib.qwn_x_lora_add(self.pkg.lora_array([w["rec"] for w in self.lora]), ys, ys, 3, self.dx.ptr, self.dids.ptr,
                                  self.T) == 0

    def append(self, lib):
        q, k, v = self.qkv
        assert lib.qwn_x_kv_append(C.byref(self.b.cache), C.byref(self.b.batch), C.byref(self.rope), q.ptr, self.rows[0],
                                   self.heads, self.q.ptr, k.ptr, self.rows[1], v.ptr, self.rows[2]) == 0

    def attend(self, lib):
        assert lib.qwn_x_attn_paged(C.byref(self.b.cache), C.byref(self.b.batch), self.q.ptr, self.heads, 0.125, self.o.ptr,
                                    self.rows[0], 0) == 0

    def out(self, lib):
        lib.qwn_x_quantize_act_chunk(self.o.ptr, self.rows[0], self.T, self.aq.ptr, self.as_.ptr, self.asum.ptr)
        assert lib.qwn_x_gemm_w4a8(self.wo.ref, self.aq.ptr, self.as_.ptr, self.asum.ptr, self.y.ptr, self.T, None, 0) == 0
        y = ref.ptrs([self.y])
        assert lib.qwn_x_lora_add(self.pkg.lora_array([self.lora_o["rec"]]), y, y, 1, self.o.ptr, self.dids.ptr, self.T) == 0

    def all(self, lib):
        for stage in (self.project, self.adapt, self.append, self.attend, self.out):
            stage(lib)


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("lens", [[(1, 30), (1, 1), (1, 100), (1, 17), (1, 64), (1, 16), (1, 3), (1, 250)],
                                  [(37, 90), (1, 200), (50, 50)]], ids=["decode", "chunks"])
def test_attention_layer(lib, pkg, wl, lens, e4m3):
    m = Layer(pkg, wl, lens, e4m3, seed=len(lens))
    m.upload()
    T, f32 = m.T, torch.float32

    def got(bufs, widths):
        lib.tq_sync()
        return [ref.down(b, f32, (T, w)) for b, w in zip(bufs, widths)]

    m.project(lib)
    base = got(m.qkv, m.rows)
    m.adapt(lib)
    qkv = got(m.qkv, m.rows)
    for y, y0, w in zip(qkv, base, m.lora):          # a sum of 320 and one of 16 products, in fp32
        want = ref.lora(m.x, m.ids, w["a"], w["b"], None, None, y0)
        size = ref.lora(m.x.abs(), m.ids, w["a"].abs(), w["b"].abs(), None, None, y0.abs())
        assert ((y.double() - want).abs() <= size * 64 * 2.0 ** -24).all()
    m.append(lib)
    lib.tq_sync()
    q = ref.down(m.q, torch.bfloat16, (T, m.heads, m.dim))
    wq, wk, wv = ref.append(m.b, torch.cat(qkv, 1), m.heads, m.inv, 32, False, m.qn, m.kn)
    assert ((q.double() - wq).abs() <= wq.abs() * 2.0 ** -8 + 2.0 ** -16).all()
    shape = (m.b.pages, m.kv, m.b.page_size, m.dim)
    for pool, dev, want, scale in ((m.b.k, m.b.dk, wk, m.b.k_scale), (m.b.v, m.b.dv, wv, m.b.v_scale)):
        new = ref.down(dev, m.b.dtype, shape)
        step, floor = (2.0 ** -4, 2.0 ** -10) if e4m3 else (2.0 ** -8, 2.0 ** -16)
        assert ((new.double() - want.clamp(-448, 448) if e4m3 else new.double() - want).abs() <= want.abs() * step + floor).all()
        pool.copy_(new)                              # what the attention reads
    m.attend(lib)
    o = got([m.o], m.rows[:1])[0]
    top = max(m.b.k.float().abs().max(), m.b.v.float().abs().max()).double()
    assert ((o.double() - ref.attention(m.b, q, 2, 0.125)).abs() <= top * 2.0 ** -15).all()
    m.out(lib)
    y = got([m.y], [m.hidden])[0]
    assert torch.isfinite(y).all() and lib.tq_last_error() == 0
    # the whole layer from the projection on, captured and replayed: the same bits
    assert lib.tq_graph_capture_begin() == 0
    m.all(lib)
    graph = lib.tq_graph_capture_end()
    assert graph
    m.y.fill(0xA5)
    for _ in range(2):
        lib.tq_graph_launch(graph)
    again = got([m.y], [m.hidden])[0]
    lib.tq_graph_destroy(graph)
    assert np.array_equal(ref.bits(again), ref.bits(y)) and lib.tq_last_error() == 0
