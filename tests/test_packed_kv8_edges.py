"""CPU tests of the packed and 8-bit-cache entries at the edges of what they accept."""
import ctypes
import itertools
import os
import random
import re

import pytest
import torch

import acefa


def _cache(n=64, D=64):
    k = torch.zeros((1, 1, n, D), dtype=torch.int8)
    s = torch.zeros((1, 1, -(-n // 64)))
    return acefa.Kv8Cache(k, k.clone(), s, s.clone())


def _calls():
    """Well-formed calls on CPU tensors: every argument check of the library would pass."""
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    cache, x = _cache(), torch.zeros((1, 1, 64))
    q, half = torch.zeros((1, 1, 1, 64)), torch.zeros((1, 3, 64), dtype=torch.float16)
    weight, kept = torch.zeros((1, 1, 64)), torch.zeros((1, 1, 32), dtype=torch.int32)
    return {
        "store": lambda: acefa.kv8_store(cache, x, x.clone(), i32(0)),
        "load": lambda: acefa.kv8_load(cache, i32(3)),
        "attn": lambda: acefa.kv8_attn(q, cache, i32(3), weight=weight),
        "evict": lambda: acefa.Kv8Evict(cache, weight, i32(64), _cache(32), kept, i32(0))(),
        "packed": lambda: acefa.flash_attn_packed(half, half.clone(), half.clone(), i32(0, 3)),
    }


@pytest.mark.parametrize("name", ["store", "load", "attn", "evict", "packed"])
def test_tensors_in_host_memory_never_reach_a_launch(name, monkeypatch):
    """The entries cannot tell a host address from a device address, so the binding stops before it enters them."""
    lib, entered = acefa.load_library(), []

    class Spy:
        def __getattr__(self, what):
            fn = getattr(lib, what)
            if what.endswith("workspace_bytes"):  # sizes only
                return fn
            return lambda *a: entered.append(what) or acefa.OK

    monkeypatch.setattr(acefa, "_lib", Spy())
    with pytest.raises(acefa.AcefaError, match="ACEFA_ERR_DEVICE"):
        _calls()[name]()
    assert not entered


# ------------------------------------------------------------------ packed attention: dst beside q, k and v
def _t(gtype, ne, nb, data):
    t = acefa.Tensor()
    t.type, t.data = gtype, data
    t.ne[:], t.nb[:] = list(ne) + [1], list(nb) + [nb[-1] * ne[-1]]
    return t


def _packed(q, dst, k=None, n_seq=0):
    """Status of a call of no sequences: checked like any other, and never launched."""
    far = _t(acefa.GGML_F16, (64, k.ne[1] if k else 8, 1), (2, 128, 1024), 1 << 40)
    R, P = ctypes.byref, ctypes.c_void_p(256)
    return acefa.load_library().acefa_flash_attn_packed(R(q), R(k or far), R(far), R(dst), P, None, n_seq, 0, 0, 0.1, None)


ACCEPTED = (acefa.OK, -6, -7)  # the device is missing here at most
BASE = 1 << 32


def test_packed_output_on_its_operands_is_refused():
    f16, f32 = acefa.GGML_F16, acefa.GGML_F32
    D, rows, H = 64, 8, 2
    q = _t(f16, (D, rows, H), (2, 2 * D * H, 2 * D), BASE)               # (rows, H, D)
    out = lambda at, g=f16, es=2: _t(g, (D, H, rows), (es, es * D, es * D * H), at)  # noqa: E731
    size = 2 * D * H * rows
    assert _packed(q, out(BASE)) == -4                                    # in place
    assert _packed(q, out(BASE + size - 2)) == -4 and _packed(q, out(BASE - size + 2)) == -4
    assert _packed(q, out(BASE + size)) in ACCEPTED and _packed(q, out(BASE - size)) in ACCEPTED
    assert _packed(q, out(BASE - size, f32, 4)) == -4
    k = _t(f16, (D, rows, 1), (2, 2 * D, 2 * D * rows), BASE)
    far_q = _t(f16, (D, rows, H), (2, 2 * D * H, 2 * D), 1 << 41)
    assert _packed(far_q, out(BASE + 2 * D * rows - 16), k=k) == -4       # on the last key


def test_packed_output_in_one_buffer_with_its_operands():
    """Rows of [q heads | k head | output heads | more]: apart, row by row; shifted by an element they meet."""
    f16 = acefa.GGML_F16
    D, rows, H = 64, 8, 2
    for step in (2 * D * (2 * H + 1), 2 * D * (2 * H + 4)):
        q = _t(f16, (D, rows, H), (2, step, 2 * D), BASE)
        k = _t(f16, (D, rows, 1), (2, step, step * rows), BASE + 2 * D * H)
        at = BASE + 2 * D * (H + 1)
        for shift, want in ((0, ACCEPTED), (-2, (-4,)), (step - 2 * D * (2 * H + 1) + 2, (-4,)), (step, (-4,))):
            dst = _t(f16, (D, H, rows), (2, 2 * D, step), at + shift)
            if shift == step:  # a row further on: still apart from q and k
                want = ACCEPTED
            assert _packed(q, dst, k=k) in want, (step, shift)
    # heads outermost, every row followed by its output
    q = _t(f16, (D, rows, H), (2, 4 * D, 4 * D * rows), BASE)
    assert _packed(q, _t(f16, (D, H, rows), (2, 4 * D * rows, 4 * D), BASE + 2 * D)) in ACCEPTED
    assert _packed(q, _t(f16, (D, H, rows), (2, 4 * D * rows, 4 * D), BASE + 2 * D - 2)) == -4


def test_packed_output_of_any_layout_against_every_address():
    """Where rows are the same distance apart the answer is that of comparing every element's address."""
    f16, r = acefa.GGML_F16, random.Random(5)
    D, seen = 64, {True: 0, False: 0}
    for _ in range(400):
        unit = 2 * D
        rows, kv_rows, H, Hkv = r.choice([1, 2, 5]), r.choice([1, 2, 7]), r.choice([1, 2, 4]), 1
        step = unit * r.choice([6, 9, 12]) + r.choice([0, 16])
        head = unit * r.choice([1, 2]) if r.random() < 0.6 else step * max(rows, kv_rows) + 16 * r.randrange(4)
        q = _t(f16, (D, rows, H), (2, step, head), BASE)
        k = _t(f16, (D, kv_rows, Hkv), (2, step, step * kv_rows), BASE + 16 * r.randrange(-60, 200))
        # rows of dst, its heads behind one another or rows apart
        d_head = unit if rows > 1 or r.random() < 0.5 else 3 * unit
        dst = _t(f16, (D, H, rows), (2, d_head, step), BASE + 16 * r.randrange(-100, 400))
        if rows > 1 and step < d_head * H:
            continue
        taken = set()
        for t in (q, k):
            for i, j in itertools.product(range(t.ne[1]), range(t.ne[2])):
                a = t.data + i * t.nb[1] + j * t.nb[2]
                taken.update(range(a, a + unit, 2))
        meets = any(x in taken for i, j in itertools.product(range(rows), range(H))
                    for x in range(dst.data + i * step + j * d_head, dst.data + i * step + j * d_head + unit, 2))
        got = _packed(q, dst, k=k)
        assert (got == -4) == meets and (meets or got in ACCEPTED), (rows, kv_rows, H, step, head)
        seen[meets] += 1
    assert min(seen.values()) > 50


# ------------------------------------------------------------------ launches beside the previous kernel
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "acestep.cpp_b200", "csrc")


@pytest.mark.parametrize("name", ["fa_packed.cu", "kv8_attn.cu", "kv8_cache.cu", "kv8_evict.cu", "kv8_internal.h"])
def test_kernels_set_up_early_read_nothing_as_constant(name):
    """They run while the previous kernel may still write their inputs and wait for its end; a read-only load
    (__ldg, ld.global.nc, a const __restrict__ argument) says that its data does not change in all that time."""
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert not re.search(r"__ldg\s*\(|ld\.global[.\w]*\.nc|__restrict__", code)
