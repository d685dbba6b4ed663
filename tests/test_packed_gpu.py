"""GPU tests of packed-sequence attention (acefa_flash_attn_packed) against the
plain 64-bit statement of kv8_ref.py.

Tolerance.  Q, K and V enter the products exactly; scores are F32 sums.  The
weights are rounded to the operands' type before the product with V: each is off
by at most u = eps / 2 of that type relative to itself, so a mean of V under
them by at most u * max|v|; F32 arithmetic (the score's sum of D products,
at most 2^-17 * A absolute with A = scale * max_ij sum_d |q_d k_d|, and the
exponential) adds 2 * (2^-17 * A + 2^-20) * max|v|; the output's own rounding adds
half a step of its type.
"""
import numpy as np
import pytest
import torch

import acefa
import kv8_ref as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cu(lens, start=0):
    return np.concatenate([[0], np.cumsum(lens)]) + start


def _inputs(seed, Hq, H, rows_q, rows_kv, D, kind):
    r = np.random.default_rng(seed)
    q = torch.from_numpy(r.standard_normal((Hq, rows_q, D)).astype(np.float32)).to(DT[kind])
    k, v = (torch.from_numpy(r.standard_normal((H, rows_kv, D)).astype(np.float32)).to(DT[kind]) for _ in range(2))
    return q, k, v


def _check(got, q, k, v, cu_q, cu_k, mask, window, scale, kind, out_kind):
    qn, kn, vn = (x.double().numpy() for x in (q, k, v))
    want = ref.packed(qn, kn, vn, cu_q, cu_k, mask, window, scale)
    on = ~np.isnan(want).any((1, 2))
    top = float(np.abs(vn).max(initial=0.0))
    A = abs(scale) * float(np.abs(qn).max((0, 1), initial=0.0) @ np.abs(kn).max((0, 1), initial=0.0))
    tol = (torch.finfo(DT[kind]).eps / 2 + 2 * (2.0 ** -17 * A + 2.0 ** -20)) * top
    g = got.double().cpu().numpy()
    err = np.abs(g[on] - want[on])
    assert (err <= tol + torch.finfo(DT[out_kind]).eps / 2 * np.abs(want[on])).all(), (err.max(initial=0), tol)
    return on, want


def _rows(total, Hq, D, many):
    """Rows of the tensors: more than the sequences have select the kernel for many rows (the few-rows kernel
    takes rows x heads x D up to 768000)."""
    return max(total, 768000 // (Hq * D) + 1) if many else total


CASES = [
    ([1], 1, 1, 64), ([1, 1, 1], 2, 1, 128), ([128], 4, 2, 128), ([127, 129, 1, 0, 64], 4, 2, 128),
    ([300, 77], 3, 1, 64), ([5] * 40, 2, 2, 64), ([513, 256, 2], 8, 1, 128), ([640], 5, 5, 128),
    ([0, 0, 200, 0], 6, 2, 64), ([1000, 30], 2, 1, 128), ([33, 255, 257, 384, 385], 4, 4, 64),
]


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("mask,window", [(0, 0), (1, 0), (2, 0), (2, 63), (2, 300)])
@pytest.mark.parametrize("kind,out_kind", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("lens,Hq,H,D", CASES)
def test_packed(lens, Hq, H, D, kind, out_kind, mask, window, many):
    total = sum(lens)
    rows = _rows(total, Hq, D, many)
    q, k, v = _inputs([len(lens), total, D], Hq, H, rows, rows, D, kind)
    cu = _cu(lens)
    out = torch.full((rows, Hq, D), 9.0, dtype=DT[out_kind], device="cuda")
    acefa.flash_attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32(cu.tolist()), mask=mask, window=window, out=out)
    assert acefa.last_path() == 3
    _check(out[:total], q[:, :total], k, v, cu, cu, mask, window, D ** -0.5, kind, out_kind)
    assert (out[total:] == 9.0).all()
    assert acefa.device_error() == 0


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("mask", [0, 1])
@pytest.mark.parametrize("lq,lk", [([5, 1, 130, 7], [200, 64, 130, 3]), ([1, 1], [1, 700]), ([64, 9], [0, 129]),
                                   ([300], [20])])
def test_queries_behind_a_prefix(mask, lq, lk, many):
    """Other offsets for the keys: the last rows of a longer sequence, fewer keys than queries, none at all
    (rows that see nothing are 0)."""
    D, Hq, H = 128, 4, 2
    q, k, v = _inputs([sum(lq), sum(lk)], Hq, H, _rows(sum(lq), Hq, D, many), sum(lk), D, "bf16")
    cu_q, cu_k = _cu(lq), _cu(lk)
    out = acefa.flash_attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32(cu_q.tolist()), _i32(cu_k.tolist()), mask=mask)[:sum(lq)]
    _check(out, q[:, :sum(lq)], k, v, cu_q, cu_k, mask, 0, D ** -0.5, "bf16", "bf16")
    if mask == 1 and lq == [300]:
        assert (out[:280] == 0).all() and (out[280:] != 0).any()


@pytest.mark.parametrize("rows", [420, 1200])
def test_strides_gaps_and_poison_around_the_sequences(rows):
    """Rows of a (rows, Hq + 2H, D) projection, offsets that start late and end early, NaN and infinity in every
    row that belongs to no sequence: none of it reaches the output, whose other rows stay as they were."""
    D, Hq, H = 128, 6, 2
    r = np.random.default_rng(12)
    x = torch.from_numpy(r.standard_normal((rows, Hq + 2 * H, D)).astype(np.float32)).half()
    cu = np.array([40, 171, 171, 300, 377])
    x[:40], x[377:] = float("nan"), float("inf")
    xd = x.cuda()
    q, k, v = (xd[:, a:b].transpose(0, 1) for a, b in ((0, Hq), (Hq, Hq + H), (Hq + H, Hq + 2 * H)))
    big = torch.full((rows, Hq + 1, D), 3.0, dtype=torch.float16, device="cuda")
    for mask in (0, 1):
        big.fill_(3.0)
        acefa.flash_attn_packed(q, k, v, _i32(cu.tolist()), mask=mask, out=big[:, :Hq])
        qc, kc, vc = (t.cpu() for t in (q, k, v))
        for t in (qc, kc, vc):
            t[:, :40], t[:, 377:] = 0, 0
        on, _ = _check(big[:, :Hq], qc, kc, vc, cu, cu, mask, 0, D ** -0.5, "f16", "f16")
        assert on.sum() == 377 - 40
        assert (big[:40] == 3.0).all() and (big[377:] == 3.0).all() and (big[:, Hq] == 3.0).all()


@pytest.mark.parametrize("many", [False, True])
def test_a_sequence_never_reads_its_neighbour(many):
    """NaN in every row of one sequence leaves the others bit for bit as they are."""
    D, Hq, H, lens = 64, 4, 2, [100, 50, 200]
    rows = _rows(350, Hq, D, many)
    q, k, v = _inputs([3, 3], Hq, H, rows, rows, D, "bf16")
    cu = _i32(_cu(lens).tolist())
    a = acefa.flash_attn_packed(q.cuda(), k.cuda(), v.cuda(), cu, mask=1)
    for t in (q, k, v):
        t[:, 100:150] = float("nan")
    b = acefa.flash_attn_packed(q.cuda(), k.cuda(), v.cuda(), cu, mask=1)
    assert torch.equal(a[:100], b[:100]) and torch.equal(a[150:350], b[150:350]) and torch.isnan(b[100:150]).all()


@pytest.mark.parametrize("mask", [0, 1])
def test_thousands_of_short_sequences(mask):
    lens = [(7 * i) % 5 for i in range(3000)] + [200, 0, 131]
    D, total = 64, sum(lens)
    q, k, v = _inputs([30, mask], 2, 1, total, total, D, "f16")
    cu = _cu(lens)
    out = acefa.flash_attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32(cu.tolist()), mask=mask)
    _check(out, q, k, v, cu, cu, mask, 0, D ** -0.5, "f16", "f16")


@pytest.mark.parametrize("many", [False, True])
def test_large_and_small_scales(many):
    D, lens = 128, [200, 129]
    rows = _rows(329, 2, D, many)
    q, k, v = _inputs([7, 7], 2, 1, rows, rows, D, "f16")
    cu = _cu(lens)
    for scale in (1.0, 0.3, 1e-6):
        out = acefa.flash_attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32(cu.tolist()), mask=1, scale=scale)[:329]
        _check(out, q[:, :329], k, v, cu, cu, 1, 0, scale, "f16", "f16")


@pytest.mark.parametrize("out_kind", ["f16", "f32"])
@pytest.mark.parametrize("many", [False, True])
def test_unaligned_output_rows(many, out_kind):
    """Output rows at an odd element offset and stride."""
    D, lens = 64, [140, 3]
    rows = _rows(143, 2, D, many)
    q, k, v = _inputs([8, 7], 2, 2, rows, rows, D, "f16")
    cu = _cu(lens)
    buf = torch.zeros(rows * (2 * D + 5) + 1, dtype=DT[out_kind], device="cuda")
    out = buf[1:].as_strided((rows, 2, D), (2 * D + 5, D + 1, 1))
    acefa.flash_attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32(cu.tolist()), mask=1, out=out)
    _check(out[:143], q[:, :143], k, v, cu, cu, 1, 0, D ** -0.5, "f16", out_kind)


@pytest.mark.parametrize("rows", [100, 6100])
def test_bad_offsets_are_skipped_and_reported(rows):
    D = 64
    q, k, v = _inputs([1, 9], 2, 1, rows, rows, D, "f16")
    out = torch.full((rows, 2, D), 5.0, dtype=torch.float16, device="cuda")
    cu = [0, 30, 20, rows + 100]  # decreasing, then past the rows
    acefa.flash_attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32(cu), mask=1, out=out)
    _check(out[:30], q[:, :30], k, v, np.array([0, 30]), np.array([0, 30]), 1, 0, D ** -0.5, "f16", "f16")
    assert (out[30:] == 5.0).all()
    assert acefa.device_error() == 5 and acefa.device_error() == 0


def test_empty_calls_launch_nothing():
    D = 64
    q, k, v = _inputs([1], 2, 1, 0, 0, D, "f16")
    acefa.flash_attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32([0]))
    assert acefa.last_launch_count() == 0


@pytest.mark.parametrize("rows", [400, 1600])
def test_captured_with_new_offsets(rows):
    D, Hq, H = 128, 4, 2
    q, k, v = _inputs([4, 9], Hq, H, rows, rows, D, "bf16")
    qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    cu = _i32([0, 100, 400, 400])
    call = acefa.PackedAttn(qd, kd, vd, cu, mask=1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call()
    for offsets in ([0, 100, 400, 400], [0, 1, 2, 400], [0, 250, 251, 399]):
        cu.copy_(_i32(offsets))
        graph.replay()
        torch.cuda.synchronize()
        _check(call.out[:400], q[:, :400], k, v, np.array(offsets), np.array(offsets), 1, 0, D ** -0.5, "bf16", "bf16")
