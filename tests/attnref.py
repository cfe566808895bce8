"""Plain 64-bit forms of the cache append, paged attention and low-rank adapters, and the device buffers
that their tests keep (numpy arrays on the host, the library's own allocations on the GPU)."""
import ctypes as C
import importlib
import math

import numpy as np
import torch

pkg = importlib.import_module("knivesysl-xe_b200")


def bits(t):
    """A tensor's memory as numpy, whatever its type."""
    t = t.contiguous()
    if t.dtype == torch.bfloat16:
        return t.view(torch.int16).numpy()
    if t.dtype == torch.float8_e4m3fn:
        return t.view(torch.uint8).numpy()
    return t.numpy()


def up(t):
    return pkg.DevBuf.from_numpy(bits(t))


def down(buf, dtype, shape):
    n = int(np.prod(shape))
    if dtype == torch.bfloat16:
        return torch.from_numpy(buf.to_numpy(np.int16, n)).view(torch.bfloat16).reshape(shape)
    if dtype == torch.float8_e4m3fn:
        return torch.from_numpy(buf.to_numpy(np.uint8, n)).view(torch.float8_e4m3fn).reshape(shape)
    return torch.from_numpy(buf.to_numpy(np.float32, n)).reshape(shape)


class Batch:
    """A batch over a random paged cache. lens: (new, total) of every request; `pad` rows behind the last one."""

    def __init__(self, lens, page_size, heads, dim, e4m3=False, seed=0, pad=0, spare=2, scales=(0.0625, 0.03125),
                 stale=None):
        g = self.gen = torch.Generator().manual_seed(seed)
        self.lens, self.page_size, self.heads, self.dim, self.e4m3 = lens, page_size, heads, dim, e4m3
        self.k_scale, self.v_scale = scales if e4m3 else (1.0, 1.0)
        self.start = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
        self.kv_len = np.array([t for _, t in lens], np.int32)
        need = [-(-t // page_size) for _, t in lens]
        self.pages = sum(need) + spare
        self.tokens = int(self.start[-1]) + pad
        order = torch.randperm(self.pages, generator=g).numpy().astype(np.int32)
        self.table = np.full((max(1, len(lens)), max(1, max(need, default=1))), -1, np.int32)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = order[at:at + n]
            at += n
        self.dtype = torch.float8_e4m3fn if e4m3 else torch.bfloat16
        shape = (self.pages, heads, page_size, dim)
        self.k = (torch.randn(shape, generator=g) / self.k_scale).to(self.dtype)
        self.v = (torch.randn(shape, generator=g) / self.v_scale).to(self.dtype)
        if stale is not None:           # what no request has written holds this value
            live = torch.zeros(self.pages, page_size, dtype=torch.bool)
            for r, (_, total) in enumerate(lens):
                p = np.arange(total)
                live[self.table[r, p // page_size], p % page_size] = True
            for pool in (self.k, self.v):
                wide = pool.float()
                wide[~live[:, None, :].expand(-1, heads, -1)] = stale
                pool.copy_(wide.to(self.dtype))
        self.max_new = max([n for n, _ in lens], default=0)

    def upload(self):
        self.dk, self.dv = up(self.k), up(self.v)
        self.dstart, self.dlen, self.dtable = (pkg.DevBuf.from_numpy(x) for x in (self.start, self.kv_len, self.table))
        self.cache = pkg.KvCache(self.dk.ptr, self.dv.ptr, self.pages, self.page_size, self.heads, self.dim,
                                 int(self.e4m3), self.k_scale, self.v_scale)
        self.batch = pkg.KvBatch(len(self.lens), self.tokens, self.max_new, self.table.shape[1], self.dstart.ptr,
                                 self.dlen.ptr, self.dtable.ptr)
        return self

    def rows(self, pool, r, scale):
        """The cached rows of request r: [total][heads][dim] in 64 bits."""
        p = np.arange(self.lens[r][1])
        return pool[torch.from_numpy(self.table[r, p // self.page_size]).long(), :, p % self.page_size].double() * scale


def attention(b, q, group, scale):
    """softmax(scale q k) v of every new token, in 64 bits: [tokens][q heads * dim]; padding rows are NaN."""
    out = torch.full((b.tokens, b.heads * group, b.dim), math.nan, dtype=torch.float64)
    for r, (new, total) in enumerate(b.lens):
        if not new:
            continue
        k, v = b.rows(b.k, r, b.k_scale), b.rows(b.v, r, b.v_scale)
        x = q[b.start[r]:b.start[r] + new].double().reshape(new, b.heads, group, b.dim)
        s = torch.einsum("ihgd,jhd->hgij", x, k) * scale
        hidden = torch.arange(total)[None] > torch.arange(total - new, total)[:, None]
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        # a hidden key adds nothing, whatever its value holds
        o = torch.einsum("hgij,jhd->ihgd", p, v)
        out[b.start[r]:b.start[r] + new] = o.reshape(new, -1, b.dim)
    return out.reshape(b.tokens, -1)


def append(b, qkv, q_heads, inv_freq, rot, interleaved, q_norm=None, k_norm=None, eps=1e-6):
    """(q out, k pool, v pool) in 64 bits from fp32 rows [tokens][(q + 2 kv heads) * dim]; padding rows are NaN."""
    H, Hk, D = q_heads, b.heads, b.dim
    x = qkv.double().reshape(b.tokens, H + 2 * Hk, D)
    q, k, v = x[:, :H].clone(), x[:, H:H + Hk].clone(), x[:, H + Hk:]
    pos = torch.zeros(b.tokens, dtype=torch.float64)
    for r, (new, total) in enumerate(b.lens):
        pos[b.start[r]:b.start[r] + new] = torch.arange(total - new, total, dtype=torch.float64)
    for h, w in ((q, q_norm), (k, k_norm)):
        if w is not None:
            h *= torch.rsqrt(h.square().mean(2, keepdim=True) + eps) * (1.0 + w.double())
        if rot:
            angle = pos[:, None] * inv_freq.double()
            c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
            one, two = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
            u, w2 = h[..., one].clone(), h[..., two].clone()
            h[..., one], h[..., two] = u * c - w2 * s, w2 * c + u * s
    pools = []
    for pool, rows, scale in ((b.k, k, b.k_scale), (b.v, v, b.v_scale)):
        pool = pool.double()
        for r, (new, total) in enumerate(b.lens):
            p = np.arange(total - new, total)
            pool[torch.from_numpy(b.table[r, p // b.page_size]).long(), :, p % b.page_size] = \
                rows[b.start[r]:b.start[r] + new] / scale
        pools.append(pool)
    q[b.start[-1]:] = math.nan
    return q, pools[0], pools[1]


def lora(x, adapter, a, b, rank, scale, base):
    """base + scale (x A^T) B^T in 64 bits, adapter by adapter."""
    y = base.double().clone() if base is not None else torch.zeros(x.shape[0], b.shape[1], dtype=torch.float64)
    for i in range(a.shape[0]):
        t = (adapter == i).nonzero()[:, 0]
        r = int(rank[i]) if rank is not None else a.shape[1]
        f = float(scale[i]) if scale is not None else 1.0
        y[t] += f * (x[t].double() @ a[i, :r].double().T) @ b[i, :, :r].double().T
    return y


def ptrs(bufs):
    return (C.c_void_p * len(bufs))(*[b.ptr if b is not None else None for b in bufs])
