"""GPU tests of the packed and 8-bit-cache entries at the edges of what they
accept, against the plain 64-bit statements of kv8_ref.py."""
import numpy as np
import pytest
import torch

import acefa
import kv8_ref as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LOG2E = 1.4426950408889634


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ small weights beside a large one
# Four sinks of weight 1 (the first key of every 16 of the first 64, whose values are 0) and thousands of keys
# 2^-20 .. 2^-27 below them: what the output consists of are the small weights alone.
#
# Tolerance.  A score is off by at most e absolute (below), so a weight by a factor within exp(+-e) and twice
# that after the normalisation, plus 2^-20 for the exponential and u for the weight's rounding (11 bits where
# Q and the output have 16, else 22): a share r = 2e + 2^-20 + u of the mean of |v|, which is the output, all v
# being positive; F32 sums add 2^-18 of it.  A weight that is too small for the rounding's exponents is off by
# at most 2^-32 of the largest, and there are n of them over a sum of at least 4.  The output's own rounding:
# half a step of its type, 2^-25 where F16 is subnormal.
def _sink_values(r, n, low, high):
    t = r.integers(4 * low, 4 * high + 1, n)  # quarters of a power of two
    t[[0, 16, 32, 48]] = 0
    v = r.integers(1, 128, n)
    v[[0, 16, 32, 48]] = 0
    return t, v


def _sink_want(score, v):
    p = np.exp2(score - score.max())
    return float(p @ v / p.sum())


def _sink_tol(want, n, e, u, kind):
    return (2 * e + 2.0 ** -20 + u + 2.0 ** -18) * want + n * 2.0 ** -34 + torch.finfo(DT[kind]).eps / 2 * want + 2.0 ** -25


@pytest.mark.parametrize("low,high", [(25.25, 27), (20, 27)])
@pytest.mark.parametrize("D,G,n_q,kind", [(128, 1, 1, "f32"), (64, 4, 1, "f32"), (64, 8, 1, "f32"), (64, 3, 4, "f32"),
                                          (128, 2, 1, "bf16"), (64, 16, 1, "f16"), (128, 6, 4, "bf16")])
@pytest.mark.parametrize("sets,H", [(37, 1), (40, 8)])  # a cluster per unit; units of their own CTAs
def test_small_weights_of_the_8_bit_cache(sets, H, D, G, n_q, kind, low, high):
    n = 8192
    r = np.random.default_rng([sets, D, G, n_q])
    t, v = _sink_values(r, n, low, high)
    k8 = torch.from_numpy(r.integers(-127, 128, (n, D), dtype=np.int8))  # (dims that Q does not look at)
    k8[:, 0] = torch.from_numpy(-t)
    v8 = torch.from_numpy(np.repeat(v.astype(np.int8)[:, None], D, 1))
    tile = lambda x: x.cuda().expand(sets, H, n, D).contiguous()  # noqa: E731
    scales = [torch.full((sets, H, n // 64), x, device="cuda") for x in (1.0, 1.0 / 127.0)]
    cache = acefa.Kv8Cache(tile(k8), tile(v8), *scales)
    scale = D ** -0.5
    q = torch.zeros((sets, G * H, n_q, D), dtype=DT[kind], device="cuda")
    q[..., 0] = 0.25 / (scale * LOG2E)
    out = acefa.kv8_attn(q, cache, _i32([n] * sets), scale=scale).double().cpu().numpy()
    q0 = float(q[0, 0, 0, 0])
    for iq in range(n_q):
        ln = n - (n_q - 1 - iq)
        want = _sink_want(-t[:ln] * q0 * scale * LOG2E, v[:ln] * float(np.float32(1.0 / 127.0)))
        A = scale * q0 * 4 * high
        tol = _sink_tol(want, n, (2.0 ** -21 + D / 8 * 2.0 ** -23) * A, 2.0 ** -22 if kind == "f32" else 2.0 ** -11, kind)
        assert np.abs(out[:, iq] - want).max() <= tol, (iq, np.abs(out[:, iq] - want).max(), want, tol)


@pytest.mark.parametrize("low,high", [(25.25, 27), (20, 27)])
@pytest.mark.parametrize("n,D,Hq,kind,out_kind", [(1024, 64, 2, "f16", "f32"), (1024, 128, 1, "f16", "f16"),
                                                  (8192, 64, 2, "f16", "f32"), (8192, 128, 3, "f16", "f16"),
                                                  (8192, 128, 2, "bf16", "f32"), (1000, 64, 1, "bf16", "bf16")])
def test_small_weights_of_packed_sequences(n, D, Hq, kind, out_kind, low, high):
    r = np.random.default_rng([n, D, Hq])
    t, v = _sink_values(r, n, low, high)
    scale, rows = D ** -0.5, 200
    q = torch.zeros((Hq, rows, D), dtype=DT[kind])
    q[..., 0] = 0.25 / (scale * LOG2E)
    k = torch.from_numpy(r.standard_normal((1, n, D)).astype(np.float32)).to(DT[kind])
    k[..., 0] = torch.from_numpy(-t).to(DT[kind])
    v1 = torch.from_numpy(np.repeat(v[None, :, None] / 128.0, D, 2)).to(DT[kind])
    out = acefa.PackedAttn(q.cuda(), k.cuda(), v1.cuda(), _i32([0, rows]), _i32([0, n]), scale=scale,
                           out=torch.empty((rows, Hq, D), dtype=DT[out_kind], device="cuda"))().double().cpu().numpy()
    q0 = float(q[0, 0, 0])
    want = _sink_want(k[0, :, 0].double().numpy() * q0 * scale * LOG2E, v1[0, :, 0].double().numpy())
    tol = _sink_tol(want, n, 2.0 ** -17 * scale * q0 * 4 * high, torch.finfo(DT[kind]).eps / 2, out_kind)
    assert np.abs(out - want).max() <= tol, (np.abs(out - want).max(), want, tol)


# ------------------------------------------------------------------ offsets that fall back
@pytest.mark.parametrize("rows", [512, 6100])  # few rows, many rows
@pytest.mark.parametrize("empty", [0, 31, 40, 100])  # sequences ahead, of no rows
def test_packed_sequences_behind_falling_offsets_are_left_out(rows, empty):
    """Offsets that fall and rise again would give rows to two sequences: the first keeps them, whole."""
    D, a = 64, 500
    r = np.random.default_rng([rows, empty])
    q, k, v = (torch.from_numpy(r.standard_normal((h, n, D)).astype(np.float32)).half()
               for h, n in ((2, rows), (1, 900), (1, 900)))
    out = torch.full((rows, 2, D), 5.0, dtype=torch.float16, device="cuda")
    cu_q = [0] * empty + [0, a, 0, a, a + 9]
    cu_k = [0] * empty + [0, 300, 300, 900, 900]  # (the third sequence has keys of its own)
    acefa.flash_attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32(cu_q), _i32(cu_k), out=out)
    assert acefa.device_error() == 5 and acefa.device_error() == 0
    alone = acefa.flash_attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32([0, a]), _i32([0, 300]))
    assert torch.equal(out[:a], alone[:a]) and (out[a:] == 5.0).all()
    qn, kn, vn = (x.double().numpy() for x in (q, k, v))
    want = ref.packed(qn, kn, vn, [0, a], [0, 300], 0, 0, D ** -0.5)[:a]
    A = D ** -0.5 * float(np.abs(qn).max((0, 1)) @ np.abs(kn).max((0, 1)))
    u = torch.finfo(torch.float16).eps / 2  # of the weights, and of the output
    tol = (u + 2 * (2.0 ** -17 * A + 2.0 ** -20)) * np.abs(vn).max() + u * np.abs(want)
    assert (np.abs(out[:a].double().cpu().numpy() - want) <= tol).all()


def test_packed_sequence_whose_key_offsets_fall_is_the_only_one_left_out():
    D, cu_q, cu_k = 64, [0, 10, 30, 60], [50, 40, 90, 100]
    r = np.random.default_rng(3)
    q, k, v = (torch.from_numpy(r.standard_normal((1, 100, D)).astype(np.float32)).half().cuda() for _ in range(3))
    out = torch.full((100, 1, D), 5.0, dtype=torch.float16, device="cuda")
    acefa.flash_attn_packed(q, k, v, _i32(cu_q), _i32(cu_k), out=out)
    assert acefa.device_error() == 5
    good = acefa.flash_attn_packed(q[:, 10:], k, v, _i32([0, 20, 50]), _i32([40, 90, 100]))
    assert torch.equal(out[10:60], good[:50]) and (out[:10] == 5.0).all() and (out[60:] == 5.0).all()


# ------------------------------------------------------------------ eviction beside blocks that are no number
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("side", ["k", "v"])
def test_evict_moves_rows_of_a_nan_block_unchanged_and_zeros_the_rest(D, side):
    """A block of the smaller cache that takes a row whose scale is NaN gets that scale; its rows keep their
    integers, and rows behind the length are 0 like in any other block."""
    r = np.random.default_rng([D, len(side)])
    sets, H, n, keep = 2, 2, 200, 128
    q = [r.integers(-127, 128, (sets, H, n, D), dtype=np.int8) for _ in range(2)]
    s = [r.random((sets, H, 4)).astype(np.float32) + 0.1 for _ in range(2)]
    s["kv".index(side)][:, :, 1] = np.nan
    w = r.random((sets, H, n)).astype(np.float32)
    lens = [100, 200]
    cache = acefa.Kv8Cache(*(torch.from_numpy(x).cuda() for x in (*q, *s)))
    out, kept, lo, _ = acefa.kv8_evict(cache, torch.from_numpy(w).cuda(), _i32(lens), keep, 3, 20)
    for i, (tq, ts) in enumerate(((out.k, out.k_scale), (out.v, out.v_scale))):
        wq, ws, wk, wl, _ = ref.evict(q[i], s[i], w, lens, keep, 3, 20)
        assert np.array_equal(kept.cpu().numpy(), wk) and np.array_equal(lo.cpu().numpy(), wl)
        assert np.array_equal(ts.cpu().numpy(), ws, equal_nan=True)
        assert np.array_equal(tq.cpu().numpy(), wq)


# ------------------------------------------------------------------ one buffer
@pytest.mark.parametrize("rows", [100, 3100])
def test_packed_output_beside_the_projections_in_one_buffer(rows):
    """(rows, Hq + 2 Hkv + Hq, D): the output's heads behind the row's projections."""
    D, Hq, H = 64, 4, 2
    r = np.random.default_rng(rows)
    x = torch.from_numpy(r.standard_normal((rows, 2 * Hq + 2 * H, D)).astype(np.float32)).half().cuda()
    q, k, v = (x[:, a:b].transpose(0, 1) for a, b in ((0, Hq), (Hq, Hq + H), (Hq + H, Hq + 2 * H)))
    before, cu = x.clone(), _i32([0, 37, 100])
    want = acefa.flash_attn_packed(*(t.contiguous() for t in (q, k, v)), cu, mask=1)
    acefa.flash_attn_packed(q, k, v, cu, mask=1, out=x[:, Hq + 2 * H:])
    assert torch.equal(x[:100, Hq + 2 * H:], want[:100])
    assert torch.equal(x[:, :Hq + 2 * H], before[:, :Hq + 2 * H]) and torch.equal(x[100:], before[100:])


# ------------------------------------------------------------------ a loop that goes on behind evictions
@pytest.mark.parametrize("D,keep,n_max", [(128, 100, 150), (64, 64, 130), (64, 70, 71)])
def test_decode_goes_on_in_the_evicted_cache(D, keep, n_max):
    """Steps of store + attend with weights; whenever a set is full, an eviction to a cache of the same length."""
    r = np.random.default_rng([D, keep, n_max])
    sets, H, G, evictions = 3, 2, 2, 0
    cache = acefa.Kv8Cache.empty(n_max, H, sets, D)
    weight = torch.zeros((sets, H, n_max), device="cuda")
    lens = [n_max - 2, 5, n_max - 6]  # (prompts: the second stays below keep)
    cq = [np.zeros((sets, H, n_max, D), np.int8) for _ in range(2)]
    cs = [np.zeros((sets, H, -(-n_max // 64)), np.float32) for _ in range(2)]
    cu = np.concatenate([[0], np.cumsum(lens)])
    x = [r.standard_normal((H, cu[-1], D)).astype(np.float32) for _ in range(2)]
    acefa.kv8_store(cache, *(torch.from_numpy(t).cuda() for t in x), _i32([0] * sets), _i32(cu.tolist()))
    for i in range(2):
        cq[i], cs[i] = ref.store(cq[i], cs[i], x[i], [0] * sets, cu)
    total = np.zeros((sets, H, n_max))
    for _ in range(2 * (n_max - keep) + 6 if n_max - keep < 50 else 60):
        if max(lens) == n_max:
            evictions += 1
            w32 = weight.cpu().numpy()
            cache, kept, lo, weight = acefa.kv8_evict(cache, weight, _i32(lens), keep, 2, 10, n_max=n_max)
            assert cache.k.shape[2] == n_max and weight.shape == (sets, H, n_max) and (weight[..., keep:] == 0).all()
            for i in range(2):
                cq[i], cs[i], wk, wl, ww = ref.evict(cq[i], cs[i], w32, lens, keep, 2, 10)
                cq[i] = np.pad(cq[i], ((0, 0), (0, 0), (0, n_max - keep), (0, 0)))
                cs[i] = np.pad(cs[i], ((0, 0), (0, 0), (0, -(-n_max // 64) - cs[i].shape[2])))
            assert np.array_equal(kept.cpu().numpy(), wk) and np.array_equal(weight[..., :keep].cpu().numpy(), ww)
            lens = wl.tolist()
            assert lo.tolist() == lens
            total = weight.double().cpu().numpy()
        x = [r.standard_normal((H, sets, D)).astype(np.float32) for _ in range(2)]
        acefa.kv8_store(cache, *(torch.from_numpy(t).cuda() for t in x), _i32(lens))
        for i in range(2):
            cq[i], cs[i] = ref.store(cq[i], cs[i], x[i], lens, np.arange(sets + 1))
        lens = [a + 1 for a in lens]
        qn = r.standard_normal((sets, H * G, 1, D)).astype(np.float32)
        got = acefa.kv8_attn(torch.from_numpy(qn).cuda(), cache, _i32(lens), weight=weight).double().cpu().numpy()
        k, v = ref.values(cq[0], cs[0]), ref.values(cq[1], cs[1])
        want, w = ref.attend(qn.astype(np.float64), k, v, lens, D ** -0.5)
        total += w
        # a score is off by e, a weight by 2e + 2^-20 of itself, F32 sums of V by 2^-18, of weights by 2^-24 a step
        A = D ** -0.5 * max(float(np.abs(qn[b]).reshape(-1, D).max(0) @ np.abs(k[b]).reshape(-1, D).max(0)) for b in range(sets))
        e = (2.0 ** -21 + D / 8 * 2.0 ** -23) * A
        assert np.abs(got - want).max() <= (2 * e + 2.0 ** -18) * np.abs(v).max()
    # the first set is full after 2 steps and again n_max - keep later (66 of 60 steps in the second case)
    assert acefa.device_error() == 0 and evictions >= (2 if n_max - keep < 58 else 1)
    rows = (np.arange(n_max) < np.array(lens)[:, None])[:, None]  # (64 sums of two weights at most)
    gw = weight.double().cpu().numpy()
    assert (np.abs(gw - total) <= (2 * e * 4 + 2.0 ** -20 + 128 * 2.0 ** -24) * total)[np.broadcast_to(rows, gw.shape)].all()


# ------------------------------------------------------------------ Q and output of different types
# Tolerance: a score is off by at most e = (2^-21 + D / 8 * 2^-23) * A, a weight by 2e + 2^-20 of itself, where Q and
# the output both have 16 bits by its rounding to 11 too (2^-11); sums lose 2^-18; then half a step of the output.
@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("kind,out_kind", [(a, b) for a in DT for b in DT if a != b])
@pytest.mark.parametrize("D,Hq,H,n_q,lens,n_max", [
    (128, 4, 2, 1, [300, 0, 77], 320), (64, 8, 1, 1, [130], 130), (128, 16, 1, 1, [500, 64], 512), (64, 6, 2, 5, [65, 700], 704),
    (128, 2, 1, 1, [4000], 4096), (128, 24, 1, 2, [5000], 5000), (64, 12, 1, 1, [6001, 3], 6001)])
def test_attend_with_mixed_types(D, Hq, H, n_q, lens, n_max, kind, out_kind, weigh):
    r = np.random.default_rng([D, Hq, n_q, n_max])
    sets, nb = len(lens), -(-n_max // 64)
    q8 = [r.integers(-127, 128, (sets, H, n_max, D), dtype=np.int8) for _ in range(2)]
    s = [(r.random((sets, H, nb)).astype(np.float32) + 0.5) / 64 for _ in range(2)]
    cache = acefa.Kv8Cache(*(torch.from_numpy(x).cuda() for x in (*q8, *s)))
    q = torch.from_numpy(r.standard_normal((sets, Hq, n_q, D)).astype(np.float32)).to(DT[kind])
    out = torch.empty((sets, n_q, Hq, D), dtype=DT[out_kind], device="cuda")
    weight = torch.zeros((sets, H, n_max), device="cuda") if weigh else None
    acefa.kv8_attn(q.cuda(), cache, _i32(lens), weight=weight, out=out)
    qn, k, v = q.double().numpy(), ref.values(q8[0], s[0]), ref.values(q8[1], s[1])
    want, ww = ref.attend(qn, k, v, lens, D ** -0.5)
    A = D ** -0.5 * max(float(np.abs(qn[b]).reshape(-1, D).max(0) @ np.abs(k[b]).reshape(-1, D).max(0)) for b in range(sets))
    e = (2.0 ** -21 + D / 8 * 2.0 ** -23) * A
    u = 0.0 if "f32" in (kind, out_kind) else 2.0 ** -11
    tol = (2 * e + 2.0 ** -18 + u) * np.abs(v).max() + torch.finfo(DT[out_kind]).eps / 2 * np.abs(want)
    got = out.double().cpu().numpy()
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) - tol).max()
    if weigh:
        rows = Hq // H * n_q
        gw = weight.double().cpu().numpy()
        assert (np.abs(gw - ww) <= (2 * e + 2.0 ** -20 + (rows + 1) * 2.0 ** -24) * ww).all()


# ------------------------------------------------------------------ against the K and V that were stored
@pytest.mark.parametrize("D,grow", [(64, False), (128, True)])
def test_attention_over_the_cache_against_unquantised_keys_and_values(D, grow):
    """Prompts at once, then 40 rows one by one.  A value is off by at most half a step of its scale when it is
    stored and of the new scale whenever that grows: (1 + g) / 2 times the block's last scale after g growths.  A
    score is then off by at most E = scale * sum_d |q_d| times that of K, the weights' ratios by exp(2E), and
    the output by V's own error and (exp(2E) - 1) * max|v|; the kernel adds 2^-16 of max|v| (scores below 2)."""
    r = np.random.default_rng([D, grow])
    sets, H, n_max, steps, lens = 2, 2, 320, 40, [150, 230]
    cu = np.concatenate([[0], np.cumsum(lens)])
    x = [r.standard_normal((H, cu[-1], D)).astype(np.float32) for _ in range(2)]
    cache = acefa.Kv8Cache.empty(n_max, H, sets, D)
    acefa.kv8_store(cache, *(torch.from_numpy(t).cuda() for t in x), _i32([0] * sets), _i32(cu.tolist()))
    full = [np.zeros((sets, H, n_max, D)) for _ in range(2)]
    for i in range(2):
        for b, ln in enumerate(lens):
            full[i][b, :, :ln] = x[i][:, cu[b]:cu[b + 1]]
    growths = [np.zeros((sets, H, n_max // 64)) for _ in range(2)]
    scales = lambda: [t.cpu().numpy().astype(np.float64) for t in (cache.k_scale, cache.v_scale)]  # noqa: E731
    old = scales()
    for t in range(steps):
        y = [(r.standard_normal((H, sets, D)) * (1 + 0.05 * t * grow)).astype(np.float32) for _ in range(2)]
        acefa.kv8_store(cache, *(torch.from_numpy(z).cuda() for z in y), _i32([ln + t for ln in lens]))
        new = scales()
        for i in range(2):
            for b, ln in enumerate(lens):
                full[i][b, :, ln + t] = y[i][:, b]
                blk = (ln + t) // 64
                growths[i][b, :, blk] += (new[i][b, :, blk] > old[i][b, :, blk]) & ((ln + t) % 64 != 0)
        old = new
    lens = [ln + steps for ln in lens]
    assert not grow or max(g.max() for g in growths) > 3
    off = [np.repeat((1 + growths[i]) / 2 * old[i] * (1 + 2.0 ** -20), 64, -1) for i in range(2)]
    values = [t.double().cpu().numpy() for t in acefa.kv8_load(cache, _i32(lens))]
    for i in range(2):
        for b, ln in enumerate(lens):
            assert (np.abs(values[i] - full[i])[b, :, :ln] <= off[i][b, :, :ln, None]).all()
    q = (0.1 * r.standard_normal((sets, 2 * H, 1, D))).astype(np.float32)
    got = acefa.kv8_attn(torch.from_numpy(q).cuda(), cache, _i32(lens)).double().cpu().numpy()
    want, _ = ref.attend(q.astype(np.float64), *full, lens, D ** -0.5)
    for b, ln in enumerate(lens):
        E = D ** -0.5 * np.abs(q[b]).sum(-1).max() * off[0][b, :, :ln].max()
        top = np.abs(full[1][b, :, :ln]).max() + off[1][b, :, :ln].max()
        assert np.abs(got[b] - want[b]).max() <= off[1][b, :, :ln].max() + (np.expm1(2 * E) + 2.0 ** -16) * top


def test_a_nan_scale_stays_while_rows_of_its_block_stay():
    D, r = 64, np.random.default_rng(8)
    cache = acefa.Kv8Cache.empty(128, 1, 1, D)
    x = torch.from_numpy(r.standard_normal((1, 10, D)).astype(np.float32)).cuda()
    bad = x.clone()
    bad[0, 3, 5] = float("nan")
    acefa.kv8_store(cache, bad, x, _i32([0]))
    acefa.kv8_store(cache, x * 9, x, _i32([10]))
    k, v = acefa.kv8_load(cache, _i32([20]))
    assert torch.isnan(k[0, 0, :20]).all() and not torch.isnan(v).any()
    acefa.kv8_store(cache, x, x, _i32([0]))  # the block anew: no row stays
    k, _ = acefa.kv8_load(cache, _i32([10]))
    assert not torch.isnan(k).any()


# ------------------------------------------------------------------ the same bits again
@pytest.mark.parametrize("lens,Hq,H,D,kind", [([1200, 700, 41], 6, 2, 128, "bf16"), ([70, 9, 130], 4, 4, 64, "f16"),
                                              ([65 + i for i in range(40)], 3, 1, 64, "f16")])
@pytest.mark.parametrize("mask", [0, 1, 2])
def test_packed_repeats_bit_for_bit(lens, Hq, H, D, kind, mask):
    r = np.random.default_rng([len(lens), mask])
    q, k, v = (torch.from_numpy(r.standard_normal((h, sum(lens), D)).astype(np.float32)).to(DT[kind]).cuda()
               for h in (Hq, H, H))
    call = acefa.PackedAttn(q, k, v, _i32(np.concatenate([[0], np.cumsum(lens)]).tolist()), mask=mask, window=50)
    first = call().clone()
    for _ in range(10):
        call.out.fill_(7.0)
        assert torch.equal(call(), first)


@pytest.mark.parametrize("D,Hq,H,n_q,lens,n_max,kind", [
    (128, 8, 2, 1, [700, 3, 64], 768, "f32"), (64, 16, 4, 4, [3000], 6001, "f16"), (128, 16, 1, 2, [900, 5000], 5000, "f32")])
def test_attend_with_weights_repeats_bit_for_bit(D, Hq, H, n_q, lens, n_max, kind):
    r = np.random.default_rng([D, Hq, n_max])
    sets = len(lens)
    q8 = [torch.from_numpy(r.integers(-127, 128, (sets, H, n_max, D), dtype=np.int8)).cuda() for _ in range(2)]
    s = [torch.from_numpy(r.random((sets, H, -(-n_max // 64))).astype(np.float32) / 64).cuda() for _ in range(2)]
    q = torch.from_numpy(r.standard_normal((sets, Hq, n_q, D)).astype(np.float32)).to(DT[kind]).cuda()
    weight = torch.zeros((sets, H, n_max), device="cuda")
    call = acefa.Kv8Attn(q, acefa.Kv8Cache(*q8, *s), _i32(lens), weight=weight)
    first = call().clone(), weight.clone()
    for _ in range(10):
        call.out.fill_(7.0), weight.zero_()
        call()
        assert torch.equal(call.out, first[0]) and torch.equal(weight, first[1])


def test_packed_longest_sequence():
    """2^24 keys under 200 queries: one pair of row tiles streams them all, inside the bound of every wait."""
    n, D, rows = 1 << 24, 64, 200
    g = torch.Generator(device="cuda").manual_seed(24)
    q, k, v = (torch.randn((1, m, D), device="cuda", generator=g, dtype=torch.float16) for m in (rows, n, n))
    out = acefa.PackedAttn(q, k, v, _i32([0, rows]), _i32([0, n]), scale=0.5,
                           out=torch.empty((rows, 1, D), dtype=torch.float32, device="cuda"))()
    assert acefa.device_error() == 0
    num, size, den = (torch.zeros((rows, x), dtype=torch.float64, device="cuda") for x in (D, D, 1))
    top = torch.full((rows, 1), -float("inf"), dtype=torch.float64, device="cuda")
    for a in range(0, n, 1 << 18):
        s = q[0].double() @ k[0, a:a + (1 << 18)].double().T * 0.5
        new = torch.maximum(top, s.amax(-1, keepdim=True))
        f, p = torch.exp(top - new), torch.exp(s - new)
        vv = v[0, a:a + (1 << 18)].double()
        num, size, den, top = num * f + p @ vv, size * f + p @ vv.abs(), den * f + p.sum(-1, keepdim=True), new
    want = num / den
    # weights rounded to 11 bits, scores off by 2^-17 * A, and F32 sums of 2^17 tiles in a row: 2^-24 of their running
    # magnitude each, 2^-7 of the mean of |v| in all
    A = 0.5 * float(q[0].abs().amax(0).float() @ k[0].abs().amax(0).float())
    tol = (2.0 ** -11 + 2 * (2.0 ** -17 * A + 2.0 ** -20) + 2 * 2.0 ** -7) * size / den
    assert ((out[:, 0].double() - want).abs() <= tol).all()
