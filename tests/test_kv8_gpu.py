"""GPU tests of the 8-bit block-scaled KV cache (acefa_kv8_*) against the plain
64-bit statements of kv8_ref.py.

Tolerances.  Stored integers, scales, kept rows and moved rows are exact.
Attention: a score is a sum of D products of operands kept to 22 bits, added
in F32 along D / 8 tensor-core steps that lose at most 2^-23 of the running
magnitude each, so it is off by at most e = (2^-21 + D / 8 * 2^-23) * A, with
A = scale * max_rj sum_d |q_d k_d|.  A weight is then off by a factor within
exp(+-e) times the exponential's 2^-22 and twice that after the
normalisation: 2e + 2^-20 relative.  An output is a mean of V under such
weights, kept to 22 bits, plus F32 sums: |error| <= (2e + 2^-18) * max|v|
(the mean of at most 2^13 keys in fixed trees of 16 keys per step), plus half a
step of the output's type.
"""
import numpy as np
import pytest
import torch

import acefa
import kv8_ref as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _rng(*key):
    return np.random.default_rng(list(key))


def _rows(r, *shape):
    x = r.standard_normal(shape).astype(np.float32)
    x[..., ::17] *= 6.0
    return x


def _cache(r, sets, H, n, D, n_alloc=None):
    """A cache whose rows were stored from position 0, and its numpy parts; n_alloc > n: a view of a longer one."""
    n_alloc = n_alloc or n
    q = [np.zeros((sets, H, n, D), np.int8) for _ in range(2)]
    s = [np.zeros((sets, H, -(-n // 64)), np.float32) for _ in range(2)]
    for i in range(2):
        for b in range(sets):
            x = _rows(r, H, n, D)
            qq, ss = ref.store(q[i][b:b + 1], s[i][b:b + 1], x, [0], [0, n])
            q[i][b:b + 1], s[i][b:b + 1] = qq, ss
    dev = []
    for i in range(2):
        big = torch.randint(-127, 128, (sets, H, n_alloc, D), dtype=torch.int8)
        big[:, :, :n] = torch.from_numpy(q[i])
        dev.append(big.cuda()[:, :, :n])
    cache = acefa.Kv8Cache(dev[0], dev[1], torch.from_numpy(s[0]).cuda(), torch.from_numpy(s[1]).cuda())
    return cache, q, s


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cu(lens):
    return _i32(np.concatenate([[0], np.cumsum(lens)]).tolist())


# ------------------------------------------------------------------ store / load
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pos,lens,n_max", [
    ([0], [1], 1), ([0, 0], [64, 65], 65), ([63, 64, 1], [1, 1, 130], 200), ([10, 0, 70, 5], [0, 200, 1, 59], 200),
    ([100, 3], [156, 61], 256)])
def test_store_bits(D, kind, pos, lens, n_max):
    r = _rng(D, len(kind), len(pos), n_max)
    H, sets = 3, len(pos)
    cache, q, s = _cache(r, sets, H, n_max, D, n_alloc=n_max + 5)
    total = sum(lens)
    new = [torch.from_numpy(_rows(r, H, total, D) * f).to(DT[kind]) for f in (1.7, 0.3)]
    # rows of a (rows, 2, H, D) projection: strided over heads and rows
    both = torch.stack(new, 1).permute(2, 1, 0, 3).contiguous().cuda()  # (rows, 2, H, D)
    acefa.kv8_store(cache, both[:, 0].transpose(0, 1), both[:, 1].transpose(0, 1), _i32(pos), _cu(lens))
    assert acefa.last_launch_count() == 1
    cu = np.concatenate([[0], np.cumsum(lens)])
    for i, (tq, ts) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
        wq, ws = ref.store(q[i], s[i], new[i].float().numpy(), pos, cu)
        assert np.array_equal(ts.cpu().numpy(), ws)
        assert np.array_equal(tq.cpu().numpy(), wq)
    assert acefa.device_error() == 0


def test_store_equal_counts_and_step_by_step():
    """One row per set and step without cu_rows: 150 steps equal the reference's 150 stores."""
    r = _rng(5, 1)
    H, sets, D, n_max = 2, 3, 64, 150
    cache = acefa.Kv8Cache.empty(n_max, H, sets, D)
    q = [np.zeros((sets, H, n_max, D), np.int8) for _ in range(2)]
    s = [np.zeros((sets, H, 3), np.float32) for _ in range(2)]
    for t in range(n_max):
        x = [_rows(r, H, sets, D) * (1.0 + 0.3 * t) for _ in range(2)]  # the scale keeps growing
        acefa.kv8_store(cache, torch.from_numpy(x[0]).cuda(), torch.from_numpy(x[1]).cuda(), _i32([t] * sets))
        for i in range(2):
            q[i], s[i] = ref.store(q[i], s[i], x[i], [t] * sets, np.arange(sets + 1))
    assert np.array_equal(cache.k.cpu().numpy(), q[0]) and np.array_equal(cache.v.cpu().numpy(), q[1])
    assert np.array_equal(cache.k_scale.cpu().numpy(), s[0]) and np.array_equal(cache.v_scale.cpu().numpy(), s[1])


def test_store_ties_zeros_and_tiny_values():
    """Quotients that are exactly half-integers, or next to one, blocks of zeros, and subnormal scales."""
    D, H = 128, 1
    d = np.float32(0.37)
    x = np.zeros((H, 5 * 64, D), np.float32)
    half = (np.arange(127, dtype=np.float32) + np.float32(0.5)) * d  # rounded products around the ties
    x[0, 0, :127], x[0, 1, :127], x[0, 2, :127] = half, np.nextafter(half, 0), np.nextafter(half, np.inf)
    x[0, 0, 127] = np.float32(127) * d
    x[0, 64, :127], x[0, 64, 127] = np.arange(127) + 0.5, 127.0  # d = 1: exact ties
    x[0, 192] = np.float32(1e-45) * np.arange(128)               # subnormal
    x[0, 256] = np.linspace(-3e38, 3e38, 128).astype(np.float32)
    n = x.shape[1]
    cache = acefa.Kv8Cache.empty(n, H, 1, D)
    acefa.kv8_store(cache, torch.from_numpy(x).cuda(), torch.from_numpy(-x).cuda(), _i32([0]))
    for sign, tq, ts in ((1, cache.k, cache.k_scale), (-1, cache.v, cache.v_scale)):
        wq, ws = ref.store(np.zeros((1, H, n, D), np.int8), np.zeros((1, H, 5), np.float32), sign * x, [0], [0, n])
        assert np.array_equal(ts.cpu().numpy(), ws) and np.array_equal(tq.cpu().numpy(), wq)


def test_store_nan_and_infinity_mark_their_block_only():
    D, H = 64, 2
    r = _rng(9, 9)
    x = _rows(r, H, 200, D)
    x[0, 70, 3], x[1, 130, 5] = np.nan, np.inf
    cache = acefa.Kv8Cache.empty(200, H, 1, D)
    acefa.kv8_store(cache, torch.from_numpy(x).cuda(), torch.from_numpy(x).cuda(), _i32([0]))
    k, _ = acefa.kv8_load(cache, _i32([200]))
    nan = torch.isnan(k[0]).all(-1).cpu().numpy()
    want = np.zeros((H, 200), bool)
    want[0, 64:128], want[1, 128:192] = True, True
    assert np.array_equal(nan, want)
    assert not torch.isnan(k[0]).any(-1).cpu().numpy()[~want].any()


def test_store_refuses_rows_outside_on_the_device():
    """Sets whose rows do not fit stay as they were and raise device error 5; the others are written."""
    r = _rng(4, 4)
    cache, q, s = _cache(r, 4, 1, 100, 64)
    x = _rows(r, 1, 12, 64)
    pos, cu = [98, -1, 40, 0], [0, 3, 6, 9, 12]
    acefa.kv8_store(cache, torch.from_numpy(x).cuda(), torch.from_numpy(x).cuda(), _i32(pos), _i32(cu))
    wq, ws = ref.store(q[0], s[0], x, pos, cu)
    assert np.array_equal(cache.k.cpu().numpy(), wq) and np.array_equal(cache.k_scale.cpu().numpy(), ws)
    assert not np.array_equal(wq, q[0]) and np.array_equal(wq[:2], q[0][:2])
    assert acefa.device_error() == 5
    cu = [0, 3, 2, 13, 14]  # decreasing, then past the rows
    acefa.kv8_store(cache, torch.from_numpy(x).cuda(), torch.from_numpy(x).cuda(), _i32([0] * 4), _i32(cu))
    wq, ws = ref.store(wq, ws, x, [0] * 4, cu)
    assert np.array_equal(cache.k.cpu().numpy(), wq)
    assert acefa.device_error() == 5 and acefa.device_error() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_load(D, kind):
    r = _rng(D, 77, len(kind))
    cache, q, s = _cache(r, 4, 2, 130, D)
    lens, n = [0, 130, 65, 999], 100
    big = [torch.full((4, 2, n + 3, D + 4), 7.0, dtype=DT[kind], device="cuda") for _ in range(2)]
    k, v = (b[:, :, :n, 1:D + 1] if kind == "f32" else b[:, :, :n, :D] for b in big)  # f32: rows off 16 bytes
    acefa.Kv8Load(cache, _i32(lens), k, v)()
    for t, i in ((k, 0), (v, 1)):
        want = ref.values(q[i], s[i], np.float32)[:, :, :n]
        for b, ln in enumerate(lens):
            want[b, :, ln:] = 0
        assert torch.equal(t.cpu(), torch.from_numpy(want).to(DT[kind]))
    assert (big[0][:, :, n:] == 7.0).all() and (big[0][..., D + 1:] == 7.0).all()


# ------------------------------------------------------------------ attention
def _attend_tol(q, k, v, scale, D, kind):
    A = scale * max(float(np.abs(q[b]).reshape(-1, D).max(0) @ np.abs(k[b]).reshape(-1, D).max(0))
                    for b in range(q.shape[0]))
    e = (2.0 ** -21 + D / 8 * 2.0 ** -23) * A
    return (2 * e + 2.0 ** -18) * float(np.abs(v).max()), 2 * e + 2.0 ** -20, torch.finfo(DT[kind]).eps / 2


@pytest.mark.parametrize("D,Hq,H,n_q,lens,n_max,kind", [
    (128, 16, 8, 1, [701, 688], 768, "f32"),
    (128, 8, 2, 1, [1, 0, 64, 65, 300], 300, "f32"),
    (64, 3, 3, 1, [17], 40, "f16"),
    (128, 5, 1, 1, [129, 63], 130, "bf16"),
    (64, 16, 4, 4, [500, 3, 1, 0], 512, "f16"),
    (128, 8, 1, 2, [90, 200], 201, "f32"),
    (128, 12, 4, 5, [77, 128], 128, "bf16"),
    (64, 8, 1, 8, [333], 400, "f32"),
    (128, 64, 1, 1, [260, 5], 260, "f32"),
    (128, 1, 1, 17, [40], 64, "f32"),
    (64, 32, 8, 1, [2500, 30, 1200, 64, 1, 640, 0, 128], 2560, "bf16"),
    (128, 2, 2, 1, list(range(0, 140, 2)), 140, "f32"),
    # long caches of few units, and more units than CTAs: two launches
    (128, 4, 1, 1, [4000], 4096, "f32"),
    (64, 16, 2, 1, [3000, 4100], 4200, "bf16"),
    (128, 3, 1, 3, [5000], 5000, "f32"),
    (128, 16, 1, 1, [4500], 5000, "f16"),
    (64, 6, 1, 2, [6001], 6001, "f32"),
    (64, 32, 1, 2, [300, 77], 300, "bf16"),
    (128, 32, 1, 2, [7000], 7000, "f16"),
    (64, 2, 1, 1, [(37 * i) % 131 for i in range(400)], 130, "f32"),
])
@pytest.mark.parametrize("weigh", [False, True])
def test_attend(D, Hq, H, n_q, lens, n_max, kind, weigh):
    r = _rng(D, Hq, n_q, n_max)
    cache, cq, cs = _cache(r, len(lens), H, n_max, D, n_alloc=n_max + 3)
    q = torch.from_numpy(r.standard_normal((len(lens), n_q, Hq, D)).astype(np.float32)).to(DT[kind])
    qd = q.cuda().transpose(1, 2)  # (sets, Hq, n_q, D), a view
    w0 = r.random((len(lens), H, n_max)).astype(np.float32) if weigh else None
    weight = torch.from_numpy(w0).cuda() if weigh else None
    out = acefa.kv8_attn(qd, cache, _i32(lens), weight=weight)
    assert acefa.last_path() == 4 and acefa.last_launch_count() in (1, 2)
    qn = q.float().numpy().astype(np.float64).transpose(0, 2, 1, 3)
    k, v = ref.values(cq[0], cs[0]), ref.values(cq[1], cs[1])
    want, ww = ref.attend(qn, k, v, lens, D ** -0.5)
    tol, wtol, half = _attend_tol(qn, k, v, D ** -0.5, D, kind)
    got = out.float().cpu().numpy().astype(np.float64)
    assert np.abs(got - want).max() <= tol + half * np.abs(want).max()
    for b, ln in enumerate(lens):
        if ln == 0:
            assert (got[b] == 0).all()
    if weigh:
        gw = weight.cpu().numpy().astype(np.float64)
        rows = Hq // H * n_q  # F32 sums of that many weights on top of w0
        assert np.all(np.abs(gw - (w0 + ww)) <= ww * wtol + (rows + 1) * 2.0 ** -24 * (w0 + ww))
        for b, ln in enumerate(lens):
            assert np.array_equal(weight.cpu().numpy()[b, :, ln:], w0[b, :, ln:])


def test_attend_large_scores_and_small_queries():
    """Scores that grow along the keys (the running maximum moves often), rows of zeros, of 1e-30 and of 1e4."""
    r = _rng(8, 8)
    D, n = 128, 700
    x = _rows(r, 1, n, D) * np.linspace(0.1, 8, n, dtype=np.float32)[None, :, None]
    vv = _rows(r, 1, n, D)
    cache = acefa.Kv8Cache.empty(n, 1, 1, D)
    acefa.kv8_store(cache, torch.from_numpy(x).cuda(), torch.from_numpy(vv).cuda(), _i32([0]))
    q = r.standard_normal((1, 4, 1, D)).astype(np.float32)
    q[0, 1], q[0, 2], q[0, 3] = 0.0, q[0, 2] * 1e-30, x[0, 5] * 0.4
    out = acefa.kv8_attn(torch.from_numpy(q).cuda(), cache, _i32([n])).cpu().numpy()
    k, v = (ref.values(t.cpu().numpy(), s.cpu().numpy()) for t, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    want, _ = ref.attend(q.astype(np.float64), k, v, [n], D ** -0.5)
    tol, _, half = _attend_tol(q, k, v, D ** -0.5, D, "f32")
    assert np.abs(out - want).max() <= tol + half * np.abs(want).max()


@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("D,Hq,H,n_q,sets,n_max,kind", [
    (128, 4, 4, 4, 1, 130, "f32"), (128, 8, 4, 4, 2, 130, "f32"), (64, 16, 4, 4, 1, 130, "bf16"),
    (128, 4, 1, 4, 1, 5000, "f16"), (64, 1, 1, 4, 3, 5000, "f32"), (128, 2, 1, 20, 1, 130, "f32")])
def test_a_nan_row_reaches_only_the_queries_that_see_its_block(D, Hq, H, n_q, sets, n_max, kind, side):
    """The last drafted row opens a block, and its K or V holds a NaN: the queries before it give what
    they gave without it, the last one NaN."""
    r = _rng(D, Hq, n_q, n_max, 7)
    ln = 65 + 64 * ((n_max - 66) // 64)
    cache, cq, cs = _cache(r, sets, H, n_max, D)
    bad = [_rows(r, H, sets, D) for _ in range(2)]
    bad["kv".index(side)][:, :, 3] = np.nan
    acefa.kv8_store(cache, *(torch.from_numpy(x).cuda() for x in bad), _i32([ln - 1] * sets))
    block = (ln - 1) // 64
    assert torch.isnan((cache.k_scale if side == "k" else cache.v_scale)[:, :, block]).all()
    q = torch.from_numpy(r.standard_normal((sets, Hq, n_q, D)).astype(np.float32)).to(DT[kind])
    out = acefa.kv8_attn(q.cuda(), cache, _i32([ln] * sets)).cpu()
    assert torch.isnan(out[:, -1]).all()
    # the others saw the same rows before the last one was there
    qn = q.float().numpy().astype(np.float64)
    k, v = ref.values(cq[0], cs[0]), ref.values(cq[1], cs[1])
    want, _ = ref.attend(qn[:, :, :-1], k, v, [ln - 1] * sets, D ** -0.5)
    tol, _, half = _attend_tol(qn, k, v, D ** -0.5, D, kind)
    assert np.abs(out[:, :-1].double().numpy() - want).max() <= tol + half * np.abs(want).max()


@pytest.mark.parametrize("order", ["sets", "heads", "rows"])
def test_keys_and_values_interleaved_in_one_buffer(order):
    """Store, load, attention and eviction give the bits of a cache whose K and V lie apart."""
    r = _rng(4, 5, len(order))
    D, H, sets, n, keep = 128, 2, 3, 200, 90
    lens = [200, 64, 131]
    new = [torch.from_numpy(_rows(r, H, sum(lens), D)).cuda() for _ in range(2)]
    q = torch.from_numpy(r.standard_normal((sets, 4, 1, D)).astype(np.float32)).cuda()

    def build(rows):
        scales = [torch.zeros((sets, H, -(-rows // 64)), device="cuda") for _ in range(2)]
        shape = {"sets": (sets, 2, H, rows, D), "heads": (sets, H, 2, rows, D), "rows": (sets, H, rows, 2, D)}[order]
        at = {"sets": 1, "heads": 2, "rows": 3}[order]
        both = torch.zeros(shape, dtype=torch.int8, device="cuda")
        return acefa.Kv8Cache(both.select(at, 0), both.select(at, 1), *scales)

    def run(cache, out):
        for c in (cache, out):
            for t in c.tensors:
                t.zero_()
        weight = torch.zeros((sets, H, n), device="cuda")
        kept, lo = torch.zeros((sets, H, keep), dtype=torch.int32, device="cuda"), _i32([0] * sets)
        acefa.kv8_store(cache, *new, _i32([0] * sets), _cu(lens))
        o = acefa.kv8_attn(q, cache, _i32(lens), weight=weight)
        acefa.Kv8Evict(cache, weight, _i32(lens), out, kept, lo, n_first=4, n_recent=20)()
        return [*cache.tensors, *acefa.kv8_load(cache, _i32(lens)), o, weight, *out.tensors, kept, lo]

    for a, b in zip(run(build(n), build(keep)),
                    run(acefa.Kv8Cache.empty(n, H, sets, D), acefa.Kv8Cache.empty(keep, H, sets, D))):
        assert torch.equal(a, b)


def test_attend_repeats_bit_for_bit_and_other_stream():
    r = _rng(3, 1, 4)
    cache, *_ = _cache(r, 5, 2, 900, 128)
    q = torch.from_numpy(r.standard_normal((5, 8, 1, 128)).astype(np.float32)).cuda()
    lens = _i32([900, 3, 512, 64, 777])
    call = acefa.Kv8Attn(q, cache, lens)
    first = call().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        call.out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        call(side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(call.out, first)
    got = acefa.kv8_attn(q, cache, lens, stream=side)
    side.synchronize()
    assert torch.equal(got, first)


def test_attend_captured_with_new_lengths():
    """A captured step (store + attend with weights) replays with other lengths, positions and rows."""
    r = _rng(6, 1, 4)
    D, H, sets, n_max = 128, 2, 3, 256
    cache, cq, cs = _cache(r, sets, H, n_max, D)
    q = torch.zeros((sets, 4, 1, D), device="cuda")
    new = [torch.zeros((H, sets, D), device="cuda") for _ in range(2)]
    pos, lens = _i32([0] * sets), _i32([1] * sets)
    weight = torch.zeros((sets, H, n_max), device="cuda")
    store, attend = acefa.Kv8Store(cache, new[0], new[1], pos), acefa.Kv8Attn(q, cache, lens, weight=weight)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        store(), attend()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        store(), attend()
    for i, t in enumerate((cache.k, cache.v)):
        t.copy_(torch.from_numpy(cq[i]))
    cache.k_scale.copy_(torch.from_numpy(cs[0])), cache.v_scale.copy_(torch.from_numpy(cs[1]))
    weight.zero_()
    total = np.zeros((sets, H, n_max))
    for at in ([70, 130, 255], [71, 131, 0]):
        x = [_rows(r, H, sets, D) for _ in range(2)]
        qn = r.standard_normal((sets, 4, 1, D)).astype(np.float32)
        for t, xx in zip(new, x):
            t.copy_(torch.from_numpy(xx))
        q.copy_(torch.from_numpy(qn)), pos.copy_(_i32(at)), lens.copy_(_i32([a + 1 for a in at]))
        graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            cq[i], cs[i] = ref.store(cq[i], cs[i], x[i], at, np.arange(sets + 1))
        k, v = ref.values(cq[0], cs[0]), ref.values(cq[1], cs[1])
        want, w = ref.attend(qn.astype(np.float64), k, v, [a + 1 for a in at], D ** -0.5)
        total += w
        tol, wtol, half = _attend_tol(qn, k, v, D ** -0.5, D, "f32")
        assert np.array_equal(cache.k.cpu().numpy(), cq[0]) and np.array_equal(cache.v.cpu().numpy(), cq[1])
        assert np.abs(attend.out.cpu().numpy() - want).max() <= tol + half * np.abs(want).max()
        assert np.all(np.abs(weight.cpu().numpy() - total) <= total * (2 * wtol + 2.0 ** -20))


def test_calls_side_by_side():
    """Two calls with handles of their own on two streams, on one cache."""
    r = _rng(3, 3, 3)
    cache, *_ = _cache(r, 3, 2, 3000, 64)
    lens = _i32([3000, 1, 1700])
    calls = [acefa.Kv8Attn(torch.from_numpy(r.standard_normal((3, 4, n, 64)).astype(np.float32)).cuda(), cache, lens)
             for n in (1, 3)]
    want = [c().clone() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for c, s in zip(calls, streams):
            c(s)
    torch.cuda.synchronize()
    for c, w in zip(calls, want):
        assert torch.equal(c.out, w)


def test_offsets_past_32_bits():
    """The second of two sets lies more than 4 GB behind the first: stored, read, attended, evicted."""
    r = _rng(32, 33)
    D, n, gap = 128, 200, (1 << 32) + 4096
    big = [torch.empty(gap + n * D, dtype=torch.int8, device="cuda") for _ in range(2)]
    k, v = (t.as_strided((2, 1, n, D), (gap, n * D, D, 1)) for t in big)
    scales = [torch.empty((2, 1, 4), device="cuda") for _ in range(2)]
    cache = acefa.Kv8Cache(k, v, *scales)
    x = [_rows(r, 1, 2 * n, D) for _ in range(2)]
    acefa.kv8_store(cache, torch.from_numpy(x[0]).cuda(), torch.from_numpy(x[1]).cuda(), _i32([0, 0]))
    cq, cs = zip(*[ref.store(np.zeros((2, 1, n, D), np.int8), np.zeros((2, 1, 4), np.float32), y, [0, 0], [0, n, 2 * n])
                   for y in x])
    kk, vv = acefa.kv8_load(cache, _i32([n, n]))
    assert np.array_equal(kk.cpu().numpy(), ref.values(cq[0], cs[0], np.float32))
    assert np.array_equal(vv.cpu().numpy(), ref.values(cq[1], cs[1], np.float32))
    q = r.standard_normal((2, 2, 1, D)).astype(np.float32)
    out = acefa.kv8_attn(torch.from_numpy(q).cuda(), cache, _i32([n, n - 7])).cpu().numpy()
    kn, vn = ref.values(cq[0], cs[0]), ref.values(cq[1], cs[1])
    want, _ = ref.attend(q.astype(np.float64), kn, vn, [n, n - 7], D ** -0.5)
    tol, _, half = _attend_tol(q, kn, vn, D ** -0.5, D, "f32")
    assert np.abs(out - want).max() <= tol + half * np.abs(want).max()
    _check_evict(cache, list(cq), list(cs), r.random((2, 1, n)).astype(np.float32), [n, n - 7], 90, 2, 5)


# ------------------------------------------------------------------ eviction
def _check_evict(cache, cq, cs, weight, lens, keep, n_first, n_recent):
    out, kept, lo, wo = acefa.kv8_evict(cache, torch.from_numpy(weight).cuda(), _i32(lens), keep, n_first, n_recent)
    assert acefa.last_launch_count() == 2
    for i, (tq, ts) in enumerate(((out.k, out.k_scale), (out.v, out.v_scale))):
        wq, ws, wk, wl, ww = ref.evict(cq[i], cs[i], weight, lens, keep, n_first, n_recent)
        assert np.array_equal(kept.cpu().numpy(), wk)
        assert np.array_equal(lo.cpu().numpy(), wl)
        assert np.array_equal(wo.cpu().numpy(), ww, equal_nan=True)
        assert np.array_equal(ts.cpu().numpy(), ws)
        assert np.array_equal(tq.cpu().numpy(), wq)
    return out, kept, lo, wo


@pytest.mark.parametrize("D,H,n,lens,keep,first,recent", [
    (128, 2, 300, [300, 299, 100, 0, 129], 128, 4, 30), (64, 3, 200, [200, 65], 64, 0, 0), (64, 1, 70, [70], 69, 0, 69),
    (128, 1, 1500, [1500, 1400], 700, 4, 100), (128, 1, 130, [130], 1, 0, 0), (64, 2, 100, [100, 90], 20, 10, 10),
    (64, 1, 5000, [5000, 2049], 2050, 1, 7), (64, 1, 90, [90], 200, 3, 9),
    # around the longest cache whose keys fit the registers
    (64, 1, 8192, [8192, 1025, 8161, 700], 600, 0, 3), (64, 2, 8193, [8193, 1024, 4097], 1000, 40, 0)])
def test_evict(D, H, n, lens, keep, first, recent):
    r = _rng(D, n, keep)
    cache, cq, cs = _cache(r, len(lens), H, n, D, n_alloc=n + 2)
    w = np.exp(2 * r.standard_normal((len(lens), H, n))).astype(np.float32)
    w[r.random(w.shape) < 0.3] = 0.0
    _check_evict(cache, cq, cs, w, lens, keep, first, recent)


def test_evict_more_rows_than_shared_memory_holds():
    r = _rng(50, 50)
    n, keep = 60000, 333
    q = [r.integers(-127, 128, (1, 1, n, 64), dtype=np.int8) for _ in range(2)]
    s = [r.random((1, 1, -(-n // 64))).astype(np.float32) + 0.1 for _ in range(2)]
    cache = acefa.Kv8Cache(*(torch.from_numpy(t).cuda() for t in (*q, *s)))
    w = np.exp(2 * r.standard_normal((1, 1, n))).astype(np.float32)
    w[0, 0, ::3] = w[0, 0].max()  # more equal ones than places
    _check_evict(cache, q, s, w, [n - 11], keep, 3, 4)


def test_evict_ties_and_odd_weights():
    """Equal weights go to the lower rows; -0, negative, infinite and NaN weights have their place."""
    r = _rng(2, 2)
    cache, cq, cs = _cache(r, 4, 1, 150, 64)
    w = np.zeros((4, 1, 150), np.float32)
    w[1, 0] = r.choice(np.float32([0.0, -0.0, 1.0, -1.0]), 150)
    w[2, 0] = r.choice(np.float32([np.nan, np.inf, -np.inf, 0.5, 1e-40, -1e-40]), 150)
    w[3, 0] = np.nan
    _check_evict(cache, cq, cs, w, [150, 140, 150, 150], 65, 2, 3)


def test_evict_moves_equal_scales_unchanged_and_rounds_ties_to_even():
    """Scales of a ratio of exactly 1/2 make every odd value a tie."""
    D, n = 64, 128
    q = np.tile(np.arange(-64, 64, dtype=np.int8)[:, None], (1, D))[None, None]
    s = np.float32([[[0.25, 0.5]]])
    cache = acefa.Kv8Cache(torch.from_numpy(q).cuda(), torch.from_numpy(q.copy()).cuda(), torch.from_numpy(s).cuda(),
                           torch.from_numpy(s.copy()).cuda())
    w = np.zeros((1, 1, n), np.float32)
    w[0, 0, ::2] = 1.0
    _check_evict(cache, [q, q], [s, s], w, [128], 64, 0, 0)


# ------------------------------------------------------------------ together
def test_prompt_decode_evict_decode():
    """Packed prompts, their rows into the cache, decode steps with weights, an eviction, more steps."""
    r = _rng(1, 2, 3)
    D, H, G, n_max, keep = 128, 2, 2, 256, 100
    lens = [150, 7, 64]
    total, sets = sum(lens), 3
    kk, vv = (_rows(r, H, total, D) for _ in range(2))
    qq = r.standard_normal((H * G, total, D)).astype(np.float32)
    h16 = [torch.from_numpy(x).half().cuda() for x in (qq, kk, vv)]
    cu = _cu(lens)
    out = acefa.flash_attn_packed(*h16, cu, mask=acefa.MASK_CAUSAL)
    want = ref.packed(*(x.cpu().double().numpy() for x in h16), cu.cpu().numpy(), cu.cpu().numpy(), 1, 0, D ** -0.5)
    assert np.abs(out.cpu().double().numpy() - want).max() < 4e-3 * np.abs(h16[2].cpu().numpy()).max()
    cache = acefa.Kv8Cache.empty(n_max, H, sets, D)
    acefa.kv8_store(cache, h16[1], h16[2], _i32([0] * sets), cu)
    cq = [np.zeros((sets, H, n_max, D), np.int8) for _ in range(2)]
    cs = [np.zeros((sets, H, n_max // 64), np.float32) for _ in range(2)]
    for i in range(2):
        cq[i], cs[i] = ref.store(cq[i], cs[i], h16[1 + i].float().cpu().numpy(), [0] * sets, cu.cpu().numpy())
    weight = torch.zeros((sets, H, n_max), device="cuda")
    total_w, at = np.zeros((sets, H, n_max)), list(lens)
    for step in range(12):
        if step == 6:
            small, kept, lo, wo = acefa.kv8_evict(cache, weight, _i32(at), keep, 2, 10)
            w32 = weight.cpu().numpy()
            for i in range(2):
                cq[i], cs[i], wk, wl, _ = ref.evict(cq[i], cs[i], w32, at, keep, 2, 10)
                pad = n_max - keep
                cq[i] = np.pad(cq[i], ((0, 0), (0, 0), (0, pad), (0, 0)))
                cs[i] = np.pad(cs[i], ((0, 0), (0, 0), (0, n_max // 64 - cs[i].shape[2])))
            assert np.array_equal(kept.cpu().numpy(), wk)
            # the kept rows go back into the wide cache
            cache.k[:, :, :keep], cache.v[:, :, :keep] = small.k, small.v
            cache.k_scale[:, :, :2], cache.v_scale[:, :, :2] = small.k_scale, small.v_scale
            weight.zero_()
            weight[:, :, :keep] = wo
            total_w = weight.cpu().numpy().astype(np.float64)
            at = wl.tolist()
        x = [_rows(r, H, sets, D) for _ in range(2)]
        acefa.kv8_store(cache, torch.from_numpy(x[0]).cuda(), torch.from_numpy(x[1]).cuda(), _i32(at))
        for i in range(2):
            cq[i], cs[i] = ref.store(cq[i], cs[i], x[i], at, np.arange(sets + 1))
        at = [a + 1 for a in at]
        qn = r.standard_normal((sets, H * G, 1, D)).astype(np.float32)
        got = acefa.kv8_attn(torch.from_numpy(qn).cuda(), cache, _i32(at), weight=weight).cpu().numpy()
        k, v = ref.values(cq[0], cs[0]), ref.values(cq[1], cs[1])
        want, w = ref.attend(qn.astype(np.float64), k, v, at, D ** -0.5)
        total_w += w
        tol, wtol, half = _attend_tol(qn, k, v, D ** -0.5, D, "f32")
        assert np.abs(got - want).max() <= tol + half * np.abs(want).max()
    assert np.all(np.abs(weight.cpu().numpy() - total_w) <= total_w * (2 * wtol + 2.0 ** -18))


def test_captured_behind_copies_and_other_streams():
    """One graph of every entry behind a memset, a copy or a join of two streams; replayed with new inputs
    it gives what eager calls give."""
    r = _rng(6, 6, 6)
    D, H, sets, n, keep, total = 64, 2, 2, 150, 70, 210
    lens = _i32([150, 60])
    cu = _cu([150, 60])
    src = [torch.from_numpy(_rows(r, H, total, D)).half().cuda() for _ in range(3)]
    qkv = [torch.empty_like(x) for x in src]
    cache, small = acefa.Kv8Cache.empty(n, H, sets, D), acefa.Kv8Cache.empty(keep, H, sets, D)
    q = torch.empty((sets, 2 * H, 1, D), dtype=torch.float16, device="cuda")
    weight = torch.empty((sets, H, n), device="cuda")
    kept, lo, pos = torch.empty((sets, H, keep), dtype=torch.int32, device="cuda"), _i32([0, 0]), _i32([0, 0])
    packed = acefa.PackedAttn(*qkv, cu, mask=acefa.MASK_CAUSAL)
    store, attn = acefa.Kv8Store(cache, qkv[1], qkv[2], pos, cu), acefa.Kv8Attn(q, cache, lens, weight=weight)
    evict = acefa.Kv8Evict(cache, weight, lens, small, kept, lo, n_recent=5)
    back = [torch.empty((sets, H, keep, D), device="cuda") for _ in range(2)]
    load = acefa.Kv8Load(small, lo, *back)
    outs = (packed.out, *cache.tensors, attn.out, weight, *small.tensors, kept, lo, *back)
    side = torch.cuda.Stream()

    def run():
        main = torch.cuda.current_stream()
        for a, b in zip(qkv, src):
            a.copy_(b)
        side.wait_stream(main)
        packed(side)  # behind a fork
        for t in cache.tensors:
            t.zero_()
        store()  # behind a memset
        q.copy_(src[0][:, :2 * sets].reshape(sets, 2 * H, 1, D))
        main.wait_stream(side)
        weight.zero_()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            back[0].zero_()
        main.wait_stream(side)
        attn()  # behind a join
        evict()
        load()

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for step in range(3):
        for x in src:
            x.copy_(torch.from_numpy(_rows(r, H, total, D)).half())
        graph.replay()
        got = [t.clone() for t in outs]
        for t in outs:
            t.zero_()
        run()
        for a, b in zip(got, outs):
            assert torch.equal(a, b)
    assert acefa.device_error() == 0
