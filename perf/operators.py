"""The operators either side of the projections of a served attention layer, as measurable cases.

A decoder layer takes a batch of requests, each with one new token (decoding), a few (drafts) or a
chunk of a prompt, through three operators beside its projections:

  append  the q, k and v rows that the projections left in fp32: head norm, rotation by the token's
          position, queries out as bf16, keys and values into the pages of the cache
  attend  the new tokens' queries over each request's pages, earlier tokens included
  lora    a low-rank adapter per token, added to what one to four projections of one input gave

Every case is one of the three at a size of the benchmark's projections (hidden 5120 = 40 heads of
128, keys and values of 1024 rows = 8 heads, 10240 wide attention input, MLP 17408), or of another
head layout (24 heads of 256 over 4, 32 heads of 64 over 4).

The lengths of a batch's requests come from the case alone ("lengths" names the drawing), its values
from the seed.
"""
import ctypes as C
import importlib
import math
import random

import torch

own = False


# ------------------------------------------------------------------------------- cases
def listed():
    wide = {"heads": 40, "kv_heads": 8, "dim": 128}
    deep = {"heads": 24, "kv_heads": 4, "dim": 256}
    return [
        # one stream decoding: the smallest append, nothing but latency
        {"name": "append_1", "kind": "append", **wide, "rot": 128, "norm": False, "interleaved": False,
         "cache": "bf16", "page": 64, "count": 1, "new": 1, "context": 2000, "lengths": 1},
        # a decode batch into an 8-bit cache: head norm, a quarter of each head rotated, small pages
        {"name": "append_48_e4m3", "kind": "append", **deep, "rot": 64, "norm": True, "interleaved": False,
         "cache": "e4m3", "page": 16, "count": 48, "new": 1, "context": 16000, "lengths": 2},
        # three prompts packed into one prefill chunk
        {"name": "append_4096", "kind": "append", **wide, "rot": 128, "norm": True, "interleaved": False,
         "cache": "bf16", "page": 64, "count": 3, "new": 1400, "context": 9000, "lengths": 3},
        # one stream decoding in the middle of a conversation
        {"name": "attend_1", "kind": "attend", **wide, "cache": "bf16", "page": 64, "count": 1, "new": 1,
         "context": 1500, "out": "f32", "lengths": 4},
        # a full decode batch, contexts from a few tokens to 8192
        {"name": "attend_64", "kind": "attend", **wide, "cache": "bf16", "page": 64, "count": 64, "new": 1,
         "context": 8192, "out": "f32", "lengths": 5},
        # a few streams with long documents in an 8-bit cache
        {"name": "attend_8_long", "kind": "attend", **deep, "cache": "e4m3", "page": 16, "count": 8, "new": 1,
         "context": 65536, "out": "f32", "lengths": 6},
        # a scheduler's mixed step: some requests decode, others bring chunks; pages that end inside any tile
        {"name": "attend_mixed", "kind": "attend", **wide, "cache": "bf16", "page": 48, "count": 16, "new": 600,
         "context": 4000, "out": "f32", "lengths": 7},
        # a prefill chunk of a long prompt, half of it cached before
        {"name": "attend_4096", "kind": "attend", **wide, "cache": "bf16", "page": 64, "count": 1, "new": 4096,
         "context": 8192, "out": "bf16", "lengths": 8},
        # the key projection of one decoded token with its request's adapter
        {"name": "lora_1", "kind": "lora", "K": 5120, "M": 1024, "count": 1, "T": 1, "adapters": 4, "rank": 16,
         "lengths": 9},
        # a decode batch through gate|up, two dozen fine-tunes among the requests
        {"name": "lora_64", "kind": "lora", "K": 5120, "M": 17408, "count": 2, "T": 64, "adapters": 24, "rank": 64,
         "lengths": 10},
        # prompts of a handful of fine-tunes through the down-projection
        {"name": "lora_1000", "kind": "lora", "K": 17408, "M": 5120, "count": 1, "T": 1000, "adapters": 5, "rank": 32,
         "lengths": 11},
        # a whole prefill chunk through the attention input projection
        {"name": "lora_4096", "kind": "lora", "K": 5120, "M": 10240, "count": 1, "T": 4096, "adapters": 8, "rank": 64,
         "lengths": 12},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread evenly over the logarithm."""
    v = lo * (hi / lo) ** rng.random()
    return min(hi, max(lo, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "lora"])
    lengths = rng.randrange(1 << 20)
    if kind == "lora":
        T = _log(rng, 1, 4096)
        case = {"kind": kind, "K": _log(rng, 512, 17408, 32), "M": _log(rng, 256, 17408, 16),
                "count": rng.randint(1, 3), "T": T, "adapters": _log(rng, 1, 32), "rank": 8 * rng.randint(1, 8),
                "lengths": lengths}
        while case["T"] * (case["K"] + case["M"] * 2 * case["count"]) > 4096 * 25600:
            case["T"] = (case["T"] + 1) // 2
        return case
    dim = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 6, 8])
    case = {"kind": kind, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
            "cache": rng.choice(["bf16", "e4m3"]), "page": rng.choice([8, 16, 24, 32, 48, 64, 100, 128]),
            "lengths": lengths}
    shape = rng.choice(["decode", "drafts", "mixed", "chunk"])
    if shape == "decode":
        case |= {"count": _log(rng, 1, 96), "new": 1, "context": _log(rng, 32, 32768)}
    elif shape == "drafts":
        case |= {"count": _log(rng, 1, 48), "new": rng.randint(2, 8), "context": _log(rng, 64, 16384)}
    elif shape == "mixed":
        case |= {"count": rng.randint(3, 24), "new": _log(rng, 16, 512), "context": _log(rng, 600, 4096)}
    else:
        new = _log(rng, 33, 4096)
        case |= {"count": rng.randint(1, 2), "new": new, "context": new + _log(rng, 16, 4096)}
    # never dearer than the largest listed case: neither the cache read nor the scores
    while case["count"] * case["context"] * kv_heads * dim > 64 * 8192 * 1024:
        case["count"] = (case["count"] + 1) // 2 if case["count"] > 1 else 1
        if case["count"] == 1:
            case["context"] = max(case["new"], case["context"] // 2)
    while case["count"] * case["new"] * case["context"] * case["heads"] * dim > 4096 * 8192 * 5120:
        case["count"], case["new"] = max(1, case["count"] // 2), max(1, case["new"] // 2)
    if kind == "append":
        return case | {"rot": rng.choice([dim, dim // 2, dim // 4]), "norm": rng.random() < 0.5,
                       "interleaved": rng.random() < 0.3}
    return case | {"out": rng.choice(["f32", "bf16"])}


def _lengths(case):
    """(new tokens, cached tokens with the new ones) of every request of the batch."""
    rng = random.Random(case["lengths"])
    got = []
    for i in range(case["count"]):
        if case["new"] == 1:
            new = 1
        elif case["count"] == 1:
            new = case["new"]
        elif i == 0:
            new = case["new"]                       # one request at the bound, the others anywhere below
        elif case["new"] > 8 and case["count"] > 3 and rng.random() < 0.5:
            new = 1
        else:
            new = rng.randint(1, case["new"])
        most = case["context"]
        total = most if i == 0 else new + _log(rng, 1, max(1, most - new + 1)) - 1
        got.append((new, total))
    return got


def _adapters(case):
    """(adapter of every token, -1 for none; rank of every adapter): requests are runs of tokens, some of
    them without an adapter; ranks are multiples of 8 up to the pool's."""
    rng = random.Random(case["lengths"])
    T, ids = case["T"], []
    while len(ids) < T:
        run = 1 if T <= 64 else rng.randint(1, max(1, T // 3))
        ids += [rng.choice([-1] + list(range(case["adapters"])) * 2)] * run
    if all(a < 0 for a in ids[:T]):
        ids[0] = 0
    ranks = [case["rank"] if a == 0 else rng.randrange(8, case["rank"] + 1, 8) for a in range(case["adapters"])]
    return ids[:T], ranks


# ------------------------------------------------------------------------------ prepare
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = _generator(seed)
    s = {"case": case}

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["kind"] == "lora":
        T, K, M, n, R = case["T"], case["K"], case["M"], case["adapters"], case["rank"]
        ids, ranks = _adapters(case)
        s["adapter"], s["rank"] = _ints(ids), _ints(ranks)
        s["x"] = randn(T, K)                        # normalised hidden rows, 1% of the channels outliers
        s["x"][:, torch.randperm(K, device="cuda", generator=gen)[:max(1, K // 100)]] *= 20.0
        s["a"] = [(randn(n, R, K) / math.sqrt(K)).to(torch.bfloat16) for _ in range(case["count"])]
        s["b"] = [(randn(n, M, R) * 0.1).to(torch.bfloat16) for _ in range(case["count"])]
        s["scale"] = [torch.rand(n, device="cuda", generator=gen) + 0.5 for _ in range(case["count"])]
        s["base"] = [randn(T, M) for _ in range(case["count"])]
        s["y"] = [torch.empty_like(b) for b in s["base"]]
    else:
        lens = _lengths(case)
        H, Hk, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
        T = sum(new for new, _ in lens)
        start = [0]
        for new, _ in lens:
            start.append(start[-1] + new)
        need = [-(-total // page) for _, total in lens]
        pages, most = sum(need) + 3, max(need)
        order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
        table = torch.full((len(lens), most), -1, dtype=torch.int32, device="cuda")
        at = 0
        for r, n in enumerate(need):
            table[r, :n] = order[at:at + n]
            at += n
        s["start"], s["kv_len"], s["pages"] = _ints(start), _ints([total for _, total in lens]), table
        s["tokens"], s["most_new"] = T, max(new for new, _ in lens)
        e4m3 = case["cache"] == "e4m3"
        s["k_scale"], s["v_scale"] = (0.0625, 0.03125) if e4m3 else (1.0, 1.0)
        shape = (pages, Hk, page, D)
        dtype = torch.float8_e4m3fn if e4m3 else torch.bfloat16
        for name in ("k", "v"):
            pool = s["cache_" + name] = torch.empty(shape, dtype=dtype, device="cuda")
            for p0 in range(0, pages, 512):
                n = min(512, pages - p0)
                pool[p0:p0 + n] = (randn(n, *shape[1:]) / s[name + "_scale"]).to(dtype)
        if case["kind"] == "append":
            width = (H + 2 * Hk) * D                # the projections' rows lie in one [T][q | k | v] matrix
            s["qkv"] = randn(T, width)
            s["qkv"][:, torch.randperm(width, device="cuda", generator=gen)[:max(1, width // 100)]] *= 5.0
            s["inv_freq"] = (1e6 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64)
                                     / case["rot"])).float()
            s["q_norm"], s["k_norm"] = ((randn(D) * 0.1).to(torch.bfloat16) for _ in range(2))
            s["q_out"] = torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda")
        else:
            s["q"] = (randn(T, H, D) * 1.5).to(torch.bfloat16)
            s["scale"] = 1.0 / math.sqrt(D)
            s["out"] = torch.empty(T, H * D, dtype=torch.float32 if case["out"] == "f32" else torch.bfloat16,
                                   device="cuda")
    if own:
        _handles(s)
    torch.cuda.synchronize()      # the library has a stream of its own
    return s


def _handles(s):
    """The records that a program keeps for its cache, batch and adapters, and the call's arguments."""
    pkg = importlib.import_module("knivesysl-xe_b200")
    lib = s["lib"] = pkg.load()
    assert lib.tq_set_device(torch.cuda.current_device()) == 0
    case = s["case"]
    if case["kind"] == "lora":
        n = case["count"]
        s["ws"] = [pkg.Lora(case["adapters"], case["rank"], case["M"], case["K"], a.data_ptr(), b.data_ptr(),
                            s["rank"].data_ptr(), c.data_ptr()) for a, b, c in zip(s["a"], s["b"], s["scale"])]
        s["args"] = (pkg.lora_array(s["ws"]), (C.c_void_p * n)(*[b.data_ptr() for b in s["base"]]),
                     (C.c_void_p * n)(*[y.data_ptr() for y in s["y"]]), n, s["x"].data_ptr(),
                     s["adapter"].data_ptr(), case["T"])
        return
    D, H, Hk = case["dim"], case["heads"], case["kv_heads"]
    k = s["cache_k"]
    s["cache"] = pkg.KvCache(k.data_ptr(), s["cache_v"].data_ptr(), k.shape[0], case["page"], Hk, D,
                             int(case["cache"] == "e4m3"), s["k_scale"], s["v_scale"])
    s["batch"] = pkg.KvBatch(case["count"], s["tokens"], s["most_new"], s["pages"].shape[1], s["start"].data_ptr(),
                             s["kv_len"].data_ptr(), s["pages"].data_ptr())
    if case["kind"] == "append":
        s["rope"] = pkg.Rope(s["inv_freq"].data_ptr(), case["rot"], int(case["interleaved"]),
                             s["q_norm"].data_ptr() if case["norm"] else None,
                             s["k_norm"].data_ptr() if case["norm"] else None, 1e-6)
        x, width = s["qkv"].data_ptr(), (H + 2 * Hk) * D
        s["args"] = (C.byref(s["cache"]), C.byref(s["batch"]), C.byref(s["rope"]), x, width, H,
                     s["q_out"].data_ptr(), x + 4 * H * D, width, x + 4 * (H + Hk) * D, width)
    else:
        s["args"] = (C.byref(s["cache"]), C.byref(s["batch"]), s["q"].data_ptr(), H, s["scale"],
                     s["out"].data_ptr(), H * D, int(case["out"] == "bf16"))


# ---------------------------------------------------------------------------------- run
def run(s):
    kind = s["case"]["kind"]
    if own:
        call = {"append": "qwn_x_kv_append", "attend": "qwn_x_attn_paged", "lora": "qwn_x_lora_add"}[kind]
        rc = getattr(s["lib"], call)(*s["args"])
        if rc != 0:
            raise RuntimeError(f"{call} returned {rc}")
        if kind == "append":
            return [s["q_out"], s["cache_k"], s["cache_v"]]
        return [s["out"]] if kind == "attend" else s["y"]
    if kind == "append":
        return _append(s)
    return _attend(s) if kind == "attend" else _lora(s)


def _rows(s):
    """(request, position) of every new token."""
    new = (s["start"][1:] - s["start"][:-1]).long()
    r = torch.repeat_interleave(torch.arange(new.numel(), device="cuda"), new, output_size=s["tokens"])
    return r, s["kv_len"][r].long() - s["start"][r + 1].long() + torch.arange(s["tokens"], device="cuda")


def _append(s):
    case = s["case"]
    D, H, Hk, rot, page = case["dim"], case["heads"], case["kv_heads"], case["rot"], case["page"]
    r, pos = _rows(s)
    angle = pos.double()[:, None] * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = s["qkv"].view(-1, H + 2 * Hk, D)
    qk, v = x[:, :H + Hk], x[:, H + Hk:]
    if case["norm"]:
        weight = torch.cat((s["q_norm"].float().expand(H, D), s["k_norm"].float().expand(Hk, D)))
        qk = qk * torch.rsqrt((qk * qk).mean(2, keepdim=True) + 1e-6) * (1.0 + weight)
    if case["interleaved"]:
        a, b = qk[..., 0:rot:2], qk[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(2)
    else:
        a, b = qk[..., :rot // 2], qk[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    qk = torch.cat((turned, qk[..., rot:]), -1)
    at = s["pages"][r, pos // page].long(), pos % page
    for pool, rows, scale in ((s["cache_k"], qk[:, H:], s["k_scale"]), (s["cache_v"], v, s["v_scale"])):
        rows = rows / scale
        if case["cache"] == "e4m3":
            rows = rows.clamp(-448.0, 448.0)
        bits = pool.view(torch.uint8 if case["cache"] == "e4m3" else torch.int16)
        bits[at[0], :, at[1]] = rows.to(pool.dtype).view(bits.dtype)
    return [qk[:, :H].to(torch.bfloat16), s["cache_k"], s["cache_v"]]


def _attend(s):
    case = s["case"]
    H, Hk, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    G, n, most = H // Hk, case["count"], s["most_new"]
    r, pos = _rows(s)
    i = torch.arange(s["tokens"], device="cuda") - s["start"][r].long()
    longest = s["pages"].shape[1] * page

    def rows(pool, scale):          # [request][kv head][position][dim]
        bits = pool.view(torch.uint8 if case["cache"] == "e4m3" else torch.int16)
        got = bits[s["pages"].clamp(min=0).long()].view(pool.dtype).float() * scale
        return got.permute(0, 2, 1, 3, 4).reshape(n, Hk, longest, D)

    q = torch.zeros(n, Hk, most, G, D, device="cuda")
    q[r, :, i] = s["q"].float().view(-1, Hk, G, D)
    limit = torch.full((n, most), -1, dtype=torch.long, device="cuda")
    limit[r, i] = pos
    scores = q.view(n, Hk, most * G, D) @ rows(s["cache_k"], s["k_scale"]).transpose(2, 3)
    seen = torch.arange(longest, device="cuda") <= limit[:, :, None]
    scores = scores.mul_(s["scale"]).view(n, Hk, most, G, longest).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = scores.amax(4, keepdim=True).clamp_(min=-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(4, keepdim=True)
    o = p.view(n, Hk, most * G, longest) @ rows(s["cache_v"], s["v_scale"])
    o = o.view(n, Hk, most, G, D) / total.clamp(min=1e-30)
    return [o[r, :, i].reshape(s["tokens"], H * D).to(s["out"].dtype)]


def _lora(s):
    case = s["case"]
    n, R = case["adapters"], case["rank"]
    mine = s["adapter"][:, None] == torch.arange(n, device="cuda")
    live = torch.arange(R, device="cuda") < s["rank"][:, None]
    pick = (mine[:, :, None] & live).float()

    def one(a, b, scale, base):
        h = (s["x"] @ a.float().view(n * R, -1).T).view(-1, n, R) * pick * scale[:, None]
        return base + h.view(-1, n * R) @ b.float().permute(0, 2, 1).reshape(n * R, -1)

    return [one(*w) for w in zip(s["a"], s["b"], s["scale"], s["base"])]


# --------------------------------------------------------------------------------- work
def work(case):
    """Inputs in and results out, each once; two operations per multiply-add."""
    if case["kind"] == "lora":
        T, K, M, n = case["T"], case["K"], case["M"], case["count"]
        ids, ranks = _adapters(case)
        weights = sum(2 * ranks[a] * (K + M) for a in set(ids) if a >= 0)
        return {"bytes": 4 * T * K + n * (8 * T * M + weights),
                "flops": n * sum(2 * ranks[a] * (K + M) for a in ids if a >= 0)}
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    lens = _lengths(case)
    T = sum(new for new, _ in lens)
    kv = 1 if case["cache"] == "e4m3" else 2
    if case["kind"] == "append":
        return {"bytes": T * D * (4 * (H + 2 * Hk) + 2 * H + 2 * Hk * kv), "flops": T * D * 4 * (H + Hk)}
    seen = sum(new * total - new * (new - 1) // 2 for new, total in lens)
    cached = sum(total for _, total in lens)
    return {"bytes": 2 * cached * Hk * D * kv + T * H * D * (2 + (4 if case["out"] == "f32" else 2)),
            "flops": 4 * D * H * seen}


# ------------------------------------------------------------------------------- exact
def exact(case, seed):
    """From the definitions, request by request and head by head, in 64 bits."""
    s = prepare(case, seed)
    if case["kind"] == "lora":
        outs = []
        for a, b, scale, base in zip(s["a"], s["b"], s["scale"], s["base"]):
            y = base.double()
            for i, rank in enumerate(s["rank"].tolist()):
                rows = (s["adapter"] == i).nonzero()[:, 0]
                h = s["x"][rows].double() @ a[i, :rank].double().T
                y[rows] += scale[i].double() * (h @ b[i, :, :rank].double().T)
            outs.append(y)
        return outs
    H, Hk, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    G = H // Hk
    start, kv_len = s["start"].tolist(), s["kv_len"].tolist()
    if case["kind"] == "append":
        rot, T = case["rot"], s["tokens"]
        x = s["qkv"].double().view(T, H + 2 * Hk, D)
        q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
        pos = torch.cat([torch.arange(total - (e - b), total, device="cuda")
                         for b, e, total in zip(start, start[1:], kv_len)]).double()
        j = torch.arange(rot // 2, device="cuda")
        first, second = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + rot // 2)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           pos[:, None] * s["inv_freq"].double())[:, None]

        def head_rows(h, weight):
            if case["norm"]:
                h = h / torch.sqrt(h.square().sum(2, keepdim=True) / D + 1e-6) * (1.0 + weight.double())
            h = h.clone()
            z = torch.complex(h[..., first], h[..., second]) * turn
            h[..., first], h[..., second] = z.real, z.imag
            return h

        pools = []
        for pool, rows, scale in ((s["cache_k"], head_rows(k, s["k_norm"]), s["k_scale"]),
                                  (s["cache_v"], v, s["v_scale"])):
            pool = pool.to(torch.float32).double()
            for r, total in enumerate(kv_len):
                n = start[r + 1] - start[r]
                p = torch.arange(total - n, total, device="cuda")
                pool[s["pages"][r, p // page].long(), :, p % page] = rows[start[r]:start[r + 1]] / scale
            pools.append(pool)
        return [head_rows(q, s["q_norm"])] + pools
    out = torch.empty(s["tokens"], H, D, dtype=torch.float64, device="cuda")
    for r, total in enumerate(kv_len):
        pages = s["pages"][r, :-(-total // page)].long()
        rows = torch.arange(start[r], start[r + 1], device="cuda")
        first = total - rows.numel()
        hidden = torch.arange(total, device="cuda") > first + torch.arange(rows.numel(), device="cuda")[:, None]
        for g in range(Hk):
            k, v = (s[name][pages, g].float().double().reshape(-1, D)[:total] for name in ("cache_k", "cache_v"))
            for h in range(g * G, (g + 1) * G):
                logits = s["q"][rows, h].double() @ k.T * (s["scale"] * s["k_scale"])
                p = torch.softmax(logits.masked_fill(hidden, -math.inf), 1)
                out[rows, h] = p @ v * s["v_scale"]
    return [out.view(s["tokens"], H * D)]
