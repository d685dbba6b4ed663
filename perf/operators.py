"""Cases and plain forms of the operators around a prompt and its 8-bit KV cache.

Four operators, in the order a serving program runs them:

* ``packed``: attention of whole prompts packed behind one another, grouped heads, causal or windowed;
* ``store``: new K / V rows go into a cache held in 8 bits, one scale per 64 tokens and head (and are
  read back as the values they stand for);
* ``attend``: a few new tokens per set attend over that cache; each key's attention weight is summed up;
* ``evict``: the cache keeps the tokens of the largest summed weight.

``own`` false computes them with elementary torch operations; true calls the framework.  ``exact`` is the
definition in 64 bits.  Tensors have the framework's torch shapes (ggml's ne reversed).
"""
import math

import torch

own = False

BLOCK = 64  # tokens that share a scale
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _acefa():
    import os
    import sys

    pkg = os.path.join(os.getcwd(), "acestep.cpp_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import acefa

    return acefa


# ------------------------------------------------------------------ cases
def listed():
    return [
        # captions and tags of a few requests, encoded together: the call's latency
        {"name": "packed texts", "op": "packed", "lens": "77,1,130,12,256,33,5,64", "hq": 16, "hkv": 8, "d": 128,
         "type": "f16", "out": "f16", "mask": "causal", "window": 0},
        # the prompts of one batch of requests, different lengths, four query heads per KV head
        {"name": "packed prompts", "op": "packed", "hq": 32, "hkv": 8, "d": 128, "type": "bf16", "out": "bf16",
         "lens": "512,901,64,1024,333,750,128,1000,257,640,480,96,1023,511,300,181", "mask": "causal", "window": 0},
        # long lyric prompts
        {"name": "packed long", "op": "packed", "lens": "4096,2751,1201", "hq": 16, "hkv": 8, "d": 128, "type": "bf16",
         "out": "bf16", "mask": "causal", "window": 0},
        # an encoder with a sliding window, three query heads per KV head
        {"name": "packed window", "op": "packed", "lens": "1500,777,2048,31,600", "hq": 12, "hkv": 4, "d": 64,
         "type": "f16", "out": "f16", "mask": "window", "window": 128},
        # one new token of a request and of its unconditional twin: latency
        {"name": "store token", "op": "store", "pos": "191,100", "lens": "1,1", "n_max": 256, "hkv": 8, "d": 128},
        # eight prompts into their sets, right after the packed attention
        {"name": "store prompts", "op": "store", "pos": "0,0,0,0,512,0,100,0",
         "lens": "1024,2047,77,1500,1536,600,1301,1", "n_max": 2048, "hkv": 8, "d": 128},
        # one request and its twin, two query heads per KV head, a short cache: latency
        {"name": "attend short", "op": "attend", "lens": "701,688", "n_max": 768, "n_q": 1, "hq": 16, "hkv": 8,
         "d": 128, "type": "f32", "out": "f32", "weigh": False},
        # eight requests with their twins over caches of up to 8192 tokens
        {"name": "attend batch", "op": "attend", "hq": 32, "hkv": 8, "d": 128, "type": "bf16", "out": "bf16",
         "lens": "8192,8000,7777,8191,6500,8100,8192,5001,8192,7000,8192,8064,7936,8192,8192,4097", "n_max": 8192,
         "n_q": 1, "weigh": False},
        # the same step with the weights that eviction goes by
        {"name": "attend weighed", "op": "attend", "hq": 32, "hkv": 8, "d": 128, "type": "f32", "out": "f32",
         "lens": "2560,2048,1536,2559,1,2300,2047,900", "n_max": 2560, "n_q": 1, "weigh": True},
        # four drafted tokens of one long request checked at once
        {"name": "attend draft", "op": "attend", "lens": "30011", "n_max": 32768, "n_q": 4, "hq": 16, "hkv": 4,
         "d": 64, "type": "f16", "out": "f16", "weigh": True},
        # a request and its twin shrink to half
        {"name": "evict pair", "op": "evict", "lens": "2048,1999", "n_max": 2048, "hkv": 8, "d": 128, "keep": 1024,
         "first": 4, "recent": 256},
        # a whole batch shrinks, some sets are short enough to stay
        {"name": "evict batch", "op": "evict", "n_max": 8192, "hkv": 8, "d": 128, "keep": 4000, "first": 4,
         "recent": 1000, "lens": "8192,8000,7777,8191,4000,8100,8192,3001"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _text(values):
    return ",".join(str(v) for v in values)


def draw(rng):
    op = rng.choice(["packed", "packed", "store", "attend", "attend", "evict"])
    d = rng.choice([64, 128, 128])
    hkv = rng.choice([1, 2, 4, 8])
    if op == "packed":
        g = rng.choice([1, 2, 3, 4, 5, 8])
        top = _log(rng, 16, 4096)
        lens, room = [], 8192
        for _ in range(_log(rng, 1, 16)):
            n = min(_log(rng, 1, top), room)
            # padded scores of the plain form stay below the largest listed case's
            if n == 0 or (len(lens) + 1) * max(lens + [n]) ** 2 * hkv * g > 200e6:
                break
            lens.append(n)
            room -= n
        mask = rng.choice(["causal", "causal", "window", "none"])
        kind = rng.choice(["f16", "bf16"])
        return {"op": op, "lens": _text(lens or [top % 1000 + 1]), "hq": hkv * g, "hkv": hkv, "d": d, "type": kind,
                "out": kind, "mask": mask, "window": _log(rng, 1, 512) if mask == "window" else 0}
    sets = _log(rng, 1, 16)
    if op == "store":
        n_max = _log(rng, 64, 2048)
        pos, lens = [], []
        for _ in range(min(sets, 8)):
            n = _log(rng, 1, n_max) if rng.random() < 0.6 else 1
            pos.append(rng.randint(0, n_max - n))
            lens.append(n)
        return {"op": op, "pos": _text(pos), "lens": _text(lens), "n_max": n_max, "hkv": hkv, "d": d}
    n_max = _log(rng, 64, 32768 if op == "attend" else 8192)
    while sets * n_max > 65536:
        sets = (sets + 1) // 2
    lens = [n_max if rng.random() < 0.3 else _log(rng, 1, n_max) for _ in range(sets)]
    if op == "attend":
        kind = rng.choice(["f32", "f16", "bf16"])
        g = rng.choice([1, 2, 4, 5, 8])
        return {"op": op, "lens": _text(lens), "n_max": n_max, "n_q": rng.choice([1, 1, 1, 2, 4, 5]), "hq": hkv * g,
                "hkv": hkv, "d": d, "type": kind, "out": kind, "weigh": rng.random() < 0.5}
    keep = max(8, int(n_max * rng.uniform(0.2, 0.9)))
    return {"op": op, "lens": _text(lens), "n_max": n_max, "hkv": hkv, "d": d, "keep": keep,
            "first": rng.randint(0, 4), "recent": int(keep * rng.uniform(0.0, 0.5))}


def _ints(text):
    return [int(v) for v in text.split(",")]


# ------------------------------------------------------------------ inputs
def _rows(gen, shape, device):
    """Projected rows: normal, a few channels several times larger than the others."""
    x = torch.randn(shape, generator=gen, device=device)
    loud = 1.0 + 3.0 * (torch.rand(shape[-1], generator=gen, device=device) < 0.06)
    return x * loud


def _blocks(n):
    return -(-n // BLOCK)


def _steps(amax):
    """The scale of values up to amax: amax / 127, one rounding (a plain number as divisor would multiply)."""
    return amax / torch.full_like(amax, 127.0)


def _quantised(x):
    """Rows (..., n, D) as a cache holds them after one store: int8 and one scale per block."""
    n, nb = x.shape[-2], _blocks(x.shape[-2])
    xp = torch.nn.functional.pad(x, (0, 0, 0, nb * BLOCK - n))
    xp = xp.reshape(*x.shape[:-2], nb, BLOCK, x.shape[-1])
    scale = _steps(xp.abs().amax((-1, -2)))
    q = torch.round(xp.double() / torch.where(scale == 0, 1.0, scale)[..., None, None].double())
    q = q.reshape(*x.shape[:-2], nb * BLOCK, x.shape[-1])[..., :n, :]
    return q.to(torch.int8).contiguous(), scale.contiguous()


def _make_cache(gen, sets, hkv, n_max, d, device):
    k, ks = _quantised(_rows(gen, (sets, hkv, n_max, d), device))
    v, vs = _quantised(_rows(gen, (sets, hkv, n_max, d), device))
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}


def _place(lens, rows, device):
    """Where token t of sequence s sits among the packed rows: an index (n_seq, rows) and its validity."""
    n = torch.tensor(lens, device=device)
    start = torch.cumsum(n, 0) - n
    t = torch.arange(rows, device=device)
    valid = t[None, :] < n[:, None]
    return torch.where(valid, start[:, None] + t[None, :], 0), valid


def prepare(case, seed):
    device = "cuda"
    gen = torch.Generator(device=device).manual_seed(seed)
    lens, hkv, d = _ints(case["lens"]), case["hkv"], case["d"]
    st = {"case": case, "lens_host": lens}
    if case["op"] == "packed":
        dt, total = DTYPES[case["type"]], sum(lens)
        st["q"] = torch.randn((case["hq"], total, d), generator=gen, device=device).to(dt)
        st["k"] = _rows(gen, (hkv, total, d), device).to(dt)
        st["v"] = _rows(gen, (hkv, total, d), device).to(dt)
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        st["cu"] = torch.tensor(cu, dtype=torch.int32, device=device)
        st["out"] = torch.empty((total, case["hq"], d), dtype=DTYPES[case["out"]], device=device)
        st["place"] = _place(lens, max(lens), device)
    elif case["op"] == "store":
        pos, total = _ints(case["pos"]), sum(lens)
        st["cache"] = _make_cache(gen, len(lens), hkv, case["n_max"], d, device)
        st["k_new"] = _rows(gen, (hkv, total, d), device)
        st["v_new"] = _rows(gen, (hkv, total, d), device) * 1.5
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        st["cu"] = torch.tensor(cu, dtype=torch.int32, device=device)
        st["pos"] = torch.tensor(pos, dtype=torch.int32, device=device)
        st["lens"] = torch.tensor([p + n for p, n in zip(pos, lens)], dtype=torch.int32, device=device)
        shape = (len(lens), hkv, case["n_max"], d)
        st["k_out"], st["v_out"] = (torch.empty(shape, device=device) for _ in range(2))
    else:
        st["cache"] = _make_cache(gen, len(lens), hkv, case["n_max"], d, device)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=device)
        if case["op"] == "attend":
            dt = DTYPES[case["type"]]
            st["q"] = torch.randn((len(lens), case["hq"], case["n_q"], d), generator=gen, device=device).to(dt)
            st["out"] = torch.empty((len(lens), case["n_q"], case["hq"], d), dtype=DTYPES[case["out"]], device=device)
            st["weight"] = torch.zeros((len(lens), hkv, case["n_max"]), device=device) if case["weigh"] else None
        else:
            # weights as some hundred steps leave them: a long tail, many tokens that got next to nothing
            w = torch.randn((len(lens), hkv, case["n_max"]), generator=gen, device=device).mul(2.0).exp()
            w[torch.rand(w.shape, generator=gen, device=device) < 0.2] = 0.0
            st["weight"] = w
            sets, keep = len(lens), case["keep"]
            st["dst"] = {"k": torch.zeros((sets, hkv, keep, d), dtype=torch.int8, device=device),
                         "v": torch.zeros((sets, hkv, keep, d), dtype=torch.int8, device=device),
                         "k_scale": torch.zeros((sets, hkv, _blocks(keep)), device=device),
                         "v_scale": torch.zeros((sets, hkv, _blocks(keep)), device=device)}
            st["kept"] = torch.zeros((sets, hkv, keep), dtype=torch.int32, device=device)
            st["weight_out"] = torch.zeros((sets, hkv, keep), device=device)
            st["lens_out"] = torch.zeros(sets, dtype=torch.int32, device=device)
            st["k_out"], st["v_out"] = (torch.empty((sets, hkv, keep, d), device=device) for _ in range(2))
    if own:
        st["calls"] = _handles(st)
    return st


# ------------------------------------------------------------------ the framework's calls
def _handles(st):
    """The calls a program keeps for buffers that it uses again and again (as acefa.Op does)."""
    a, c = _acefa(), st["case"]
    if c["op"] == "packed":
        kind = {"causal": a.MASK_CAUSAL, "window": a.MASK_WINDOW, "none": 0}[c["mask"]]
        return (a.PackedAttn(st["q"], st["k"], st["v"], st["cu"], mask=kind, window=c["window"], out=st["out"]),)
    cache = a.Kv8Cache(**st["cache"])
    if c["op"] == "store":
        return (a.Kv8Store(cache, st["k_new"], st["v_new"], st["pos"], cu_rows=st["cu"]),
                a.Kv8Load(cache, st["lens"], st["k_out"], st["v_out"]))
    if c["op"] == "attend":
        return (a.Kv8Attn(st["q"], cache, st["lens"], weight=st["weight"], out=st["out"]),)
    dst = a.Kv8Cache(**st["dst"])
    return (a.Kv8Evict(cache, st["weight"], st["lens"], dst, st["kept"], st["lens_out"], weight_out=st["weight_out"],
                       n_first=c["first"], n_recent=c["recent"]),
            a.Kv8Load(dst, st["lens_out"], st["k_out"], st["v_out"]))


def run(st):
    if own:
        for call in st["calls"]:
            call()
    elif st["case"]["op"] == "packed":
        _plain_packed(st)
    elif st["case"]["op"] == "store":
        _plain_store(st)
    elif st["case"]["op"] == "attend":
        _plain_attend(st)
    else:
        _plain_evict(st)
    if st["case"]["op"] == "packed":
        return {"out": st["out"]}
    if st["case"]["op"] == "store":
        return {"k": st["k_out"], "v": st["v_out"]}
    if st["case"]["op"] == "attend":
        return {"out": st["out"], "weight": st["weight"]} if st["case"]["weigh"] else {"out": st["out"]}
    return {"k": st["k_out"], "v": st["v_out"], "kept": st["kept"], "lens": st["lens_out"],
            "weight": st["weight_out"]}


# ------------------------------------------------------------------ plain forms
def _softmax_rows(s, visible):
    """Softmax over the last axis of the visible entries; rows that see nothing are 0."""
    s = torch.where(visible, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _visible(case, n):
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :]
    if case["mask"] == "causal":
        return j <= i
    if case["mask"] == "window":
        return (i - j).abs() <= case["window"]
    return torch.ones((n, n), dtype=torch.bool, device="cuda")


def _plain_packed(st):
    c = st["case"]
    index, valid = st["place"]
    n_seq, rows = index.shape
    g = c["hq"] // c["hkv"]
    q = st["q"].float()[:, index].transpose(0, 1)                               # (n_seq, hq, rows, d)
    k = torch.where(valid[:, None, :, None], st["k"].float()[:, index].transpose(0, 1), 0.0)
    v = torch.where(valid[:, None, :, None], st["v"].float()[:, index].transpose(0, 1), 0.0)
    q = q.reshape(n_seq, c["hkv"], g * rows, c["d"])
    s = torch.matmul(q, k.transpose(-1, -2)).reshape(n_seq, c["hkv"], g, rows, rows) * c["d"] ** -0.5
    p = _softmax_rows(s, _visible(c, rows) & valid[:, None, None, None, :])
    o = torch.matmul(p.reshape(n_seq, c["hkv"], g * rows, rows), v).reshape(n_seq, c["hq"], rows, c["d"])
    st["out"].copy_(o.transpose(1, 2)[valid])


def _values(q, scale):
    """What the 8-bit rows (sets, H, n, D) stand for, in 32 bits."""
    return q.float() * scale.repeat_interleave(BLOCK, -1)[..., :q.shape[-2], None]


def _by_block(x, nb, fill):
    """(sets, H, n, ...) -> (sets, H, nb, BLOCK, ...)."""
    pad = x.new_full((*x.shape[:2], nb * BLOCK - x.shape[2], *x.shape[3:]), fill)
    return torch.cat([x, pad], 2).reshape(*x.shape[:2], nb, BLOCK, *x.shape[3:])


def _plain_store_one(q, scale, new, pos, cu):
    sets, hkv, n, d = q.shape
    nb, t = scale.shape[-1], torch.arange(n, device=q.device)
    count = (cu[1:] - cu[:-1]).long()
    first = t[None, :] - pos.long()[:, None]                                    # row among the set's new ones
    fresh = (first >= 0) & (first < count[:, None])                             # (sets, n)
    source = torch.where(fresh, cu[:-1].long()[:, None] + first, 0)
    x = torch.where(fresh[:, None, :, None], new[:, source].transpose(0, 1), 0.0)
    old = (first < 0)[:, None, :].expand(sets, hkv, n)
    any_new = _by_block(fresh[:, None, :].expand(sets, hkv, n), nb, False).any(-1)
    any_old = _by_block(old, nb, False).any(-1)
    need = _steps(_by_block(x, nb, 0.0).abs().amax((-1, -2)))
    grown = torch.where(any_new, torch.maximum(need, torch.where(any_old, scale, 0.0)), scale)
    safe = torch.where(grown == 0, 1.0, grown).double()
    row = lambda s: s.repeat_interleave(BLOCK, -1)[..., :n, None]  # noqa: E731
    moved = torch.round(q.double() * row(scale).double() / row(safe))
    moved = torch.where(row(any_new) & old[..., None], moved, q.double())
    q.copy_(torch.where(fresh[:, None, :, None], torch.round(x.double() / row(safe)), moved).to(torch.int8))
    scale.copy_(grown)


def _plain_store(st):
    c = st["cache"]
    live = (torch.arange(st["case"]["n_max"], device="cuda") < st["lens"][:, None])[:, None, :, None]
    _plain_store_one(c["k"], c["k_scale"], st["k_new"], st["pos"], st["cu"])
    _plain_store_one(c["v"], c["v_scale"], st["v_new"], st["pos"], st["cu"])
    st["k_out"].copy_(torch.where(live, _values(c["k"], c["k_scale"]), 0.0))
    st["v_out"].copy_(torch.where(live, _values(c["v"], c["v_scale"]), 0.0))


def _plain_attend(st):
    c, cache = st["case"], st["cache"]
    sets, g = len(st["lens_host"]), c["hq"] // c["hkv"]
    k, v = _values(cache["k"], cache["k_scale"]), _values(cache["v"], cache["v_scale"])
    q = st["q"].float().reshape(sets, c["hkv"], g * c["n_q"], c["d"])
    s = torch.matmul(q, k.transpose(-1, -2)).reshape(sets, c["hkv"], g, c["n_q"], c["n_max"]) * c["d"] ** -0.5
    i, j = torch.arange(c["n_q"], device="cuda")[:, None], torch.arange(c["n_max"], device="cuda")[None, :]
    visible = j < st["lens"][:, None, None] - (c["n_q"] - 1 - i)                  # (sets, n_q, n_max)
    p = _softmax_rows(s, visible[:, None, None])
    o = torch.matmul(p.reshape(sets, c["hkv"], g * c["n_q"], c["n_max"]), v)
    st["out"].copy_(o.reshape(sets, c["hq"], c["n_q"], c["d"]).transpose(1, 2))
    if c["weigh"]:
        st["weight"].add_(p.sum((2, 3)))


def _plain_evict(st):
    c, cache, dst = st["case"], st["cache"], st["dst"]
    n, keep, lens = c["n_max"], c["keep"], st["lens"].long()[:, None]
    t = torch.arange(n, device="cuda")[None, :]
    rank = st["weight"].clone()
    sure = (t < c["first"]) | (t >= lens - c["recent"]) | (lens <= keep)
    rank = torch.where(sure[:, None], math.inf, rank)
    rank = torch.where((t < lens)[:, None], rank, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    count = torch.clamp(lens, max=keep)                                         # (sets, 1)
    slot = torch.arange(min(keep, n), device="cuda")
    filled = (slot[None, :] < count)[:, None].expand(order.shape)
    order = torch.sort(torch.where(filled, order, n), -1).values
    at = torch.where(filled, order, 0)
    st["kept"].fill_(-1)
    st["kept"][..., :at.shape[-1]] = torch.where(filled, order, -1).int()
    st["lens_out"].copy_(count[:, 0].int())
    st["weight_out"].fill_(0.0)
    st["weight_out"][..., :at.shape[-1]] = torch.where(filled, torch.gather(st["weight"], -1, at), 0.0)
    for name, out in (("k", "k_out"), ("v", "v_out")):
        _plain_move(cache[name], cache[name + "_scale"], at, filled, dst[name], dst[name + "_scale"])
        st[out].copy_(torch.where((torch.arange(keep, device="cuda") < count)[:, None, :, None],
                                  _values(dst[name], dst[name + "_scale"]), 0.0))


def _plain_move(q, scale, at, filled, q_out, scale_out):
    rows = torch.gather(q, 2, at[..., None].expand(*at.shape, q.shape[-1])).double()
    was = torch.where(filled, torch.gather(scale, 2, at // BLOCK), 0.0)
    nb = scale_out.shape[-1]
    new = _by_block(was, nb, 0.0).amax(-1)
    safe = torch.where(new == 0, 1.0, new).double().repeat_interleave(BLOCK, -1)[..., :at.shape[-1]]
    moved = torch.round(rows * was.double()[..., None] / safe[..., None])
    q_out[..., :at.shape[-1], :] = torch.where(filled[..., None], moved, 0.0).to(torch.int8)
    scale_out.copy_(new)


# ------------------------------------------------------------------ work
def work(case):
    lens, hkv, d = _ints(case["lens"]), case["hkv"], case["d"]
    if case["op"] == "packed":
        pairs = 0
        for n in lens:
            if case["mask"] == "causal":
                pairs += n * (n + 1) // 2
            elif case["mask"] == "window":
                w = min(case["window"], n - 1)
                pairs += n * (2 * w + 1) - w * (w + 1)
            else:
                pairs += n * n
        return {"bytes": sum(lens) * d * 2 * (2 * case["hq"] + 2 * hkv), "flops": 4.0 * d * pairs * case["hq"]}
    if case["op"] == "store":
        rows = sum(lens) * hkv
        return {"bytes": 2 * rows * d * (4 + 1) + 2 * len(lens) * hkv * case["n_max"] * d * 4, "flops": 4.0 * rows * d}
    if case["op"] == "attend":
        size = {"f32": 4, "f16": 2, "bf16": 2}
        keys = sum(lens) * hkv
        scales = 8 * sum(_blocks(n) for n in lens) * hkv
        rows = len(lens) * case["hq"] * case["n_q"] * d
        return {"bytes": keys * (2 * d + (8 if case["weigh"] else 0)) + scales
                + rows * (size[case["type"]] + size[case["out"]]),
                "flops": 4.0 * keys * d * case["n_q"] * (case["hq"] // hkv)}
    kept = sum(min(n, case["keep"]) for n in lens) * hkv
    return {"bytes": sum(lens) * hkv * 4 + kept * (2 * d * 2 + 8) + 2 * len(lens) * hkv * case["keep"] * d * 4,
            "flops": 2.0 * kept * d}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"packed": _exact_packed, "store": _exact_store, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](
        case, st)


def _exact_rows(q, k, v, lo, hi):
    """softmax(q k^T / sqrt(D)) v of the keys lo[i] <= j < hi[i], and the weights; all in 64 bits."""
    s = torch.einsum("id,jd->ij", q, k) / math.sqrt(q.shape[-1])
    j = torch.arange(k.shape[0], device=q.device)
    s = s.masked_fill((j < lo[:, None]) | (j >= hi[:, None]), -math.inf)
    p = torch.softmax(s, -1)
    p = p.masked_fill((hi <= lo)[:, None], 0.0)
    return p @ v, p


def _exact_packed(case, st):
    q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
    g, out, at = case["hq"] // case["hkv"], torch.empty(st["out"].shape, dtype=torch.float64, device="cuda"), 0
    for n in st["lens_host"]:
        i = torch.arange(n, device="cuda")
        lo, hi = torch.zeros_like(i), torch.full_like(i, n)
        if case["mask"] == "causal":
            hi = i + 1
        elif case["mask"] == "window":
            lo, hi = (i - case["window"]).clamp(min=0), (i + case["window"] + 1).clamp(max=n)
        for h in range(case["hq"]):
            o, _ = _exact_rows(q[h, at:at + n], k[h // g, at:at + n], v[h // g, at:at + n], lo, hi)
            out[at:at + n, h] = o
        at += n
    return {"out": out}


def _exact_store(case, st):
    """Block by block: the scale covers the block's new rows and never falls below what its older rows use."""
    found = {}
    cu = st["cu"].tolist()
    for name, new in (("k", st["k_new"]), ("v", st["v_new"])):
        q, scale = st["cache"][name].double(), st["cache"][name + "_scale"].clone()
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        for s, (pos, n) in enumerate(zip(_ints(case["pos"]), st["lens_host"])):
            for b in range(_blocks(pos + n)):
                lo, hi = b * BLOCK, min(b * BLOCK + BLOCK, pos + n)
                a = max(lo, pos)  # first new row of the block
                d = scale[s, :, b]
                if a < hi:
                    x = new[:, cu[s] + a - pos:cu[s] + hi - pos]
                    need = _steps(x.abs().amax((1, 2)))
                    d_new = torch.maximum(need, d) if a > lo else need
                    div = torch.where(d_new == 0, 1.0, d_new).double()[:, None, None]
                    q[s, :, a:hi] = torch.round(x.double() / div)
                    q[s, :, lo:a] = torch.round(q[s, :, lo:a] * d.double()[:, None, None] / div)
                    d = d_new
                out[s, :, lo:hi] = q[s, :, lo:hi] * d.double()[:, None, None]
        found[name] = out
    return found


def _exact_attend(case, st):
    cache, g, n_q = st["cache"], case["hq"] // case["hkv"], case["n_q"]
    out = torch.empty(st["out"].shape, dtype=torch.float64, device="cuda")
    weight = torch.zeros((len(st["lens_host"]), case["hkv"], case["n_max"]), dtype=torch.float64, device="cuda")
    for s, n in enumerate(st["lens_host"]):
        block = torch.arange(n, device="cuda") // BLOCK
        hi = (n - (n_q - 1 - torch.arange(n_q, device="cuda"))).clamp(min=0)
        for h in range(case["hkv"]):
            k = cache["k"][s, h, :n].double() * cache["k_scale"][s, h].double()[block, None]
            v = cache["v"][s, h, :n].double() * cache["v_scale"][s, h].double()[block, None]
            for i in range(g):
                o, p = _exact_rows(st["q"][s, h * g + i].double(), k, v, torch.zeros_like(hi), hi)
                out[s, :, h * g + i] = o
                weight[s, h, :n] += p.sum(0)
    return {"out": out, "weight": weight} if case["weigh"] else {"out": out}


def _exact_evict(case, st):
    """Set by set and head by head: sort by (weight, index), keep, move."""
    keep, shape = case["keep"], st["k_out"].shape
    found = {"k": torch.zeros(shape, dtype=torch.float64, device="cuda"),
             "v": torch.zeros(shape, dtype=torch.float64, device="cuda"),
             "kept": torch.full(shape[:3], -1, dtype=torch.int32, device="cuda"),
             "lens": st["lens_out"].clone(), "weight": torch.zeros(shape[:3], dtype=torch.float64, device="cuda")}
    w = st["weight"].double().cpu().numpy()
    for s, n in enumerate(st["lens_host"]):
        m = min(n, keep)
        found["lens"][s] = m
        for h in range(case["hkv"]):
            sure = [t for t in range(n) if t < case["first"] or t >= n - case["recent"]]
            if n <= keep:
                at = list(range(n))
            else:
                rest = range(case["first"], n - case["recent"])
                rest = sorted(rest, key=lambda t: (-w[s, h, t], t))
                at = sorted(sure + rest[:keep - len(sure)])
            at = torch.tensor(at, device="cuda")
            found["kept"][s, h, :m] = at.int()
            found["weight"][s, h, :m] = st["weight"][s, h, at].double()
            for name in ("k", "v"):
                d = st["cache"][name + "_scale"][s, h][at // BLOCK].double()
                x = st["cache"][name][s, h, at].double() * d[:, None]
                for lo in range(0, m, BLOCK):
                    hi = min(m, lo + BLOCK)
                    top = d[lo:hi].max()
                    found[name][s, h, lo:hi] = torch.round(x[lo:hi] / top) * top
    return found
