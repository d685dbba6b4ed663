"""CPU tests of the refusals of acefa_kv8_* and acefa_flash_attn_packed: every
argument check answers before any device is touched."""
import ctypes

import pytest
import torch

import acefa

P = ctypes.c_void_p(256)  # an address that no check reads


@pytest.fixture(scope="module")
def lib():
    import importlib.util
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location("acestep_build", os.path.join(root, "acestep.cpp_b200", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.build()
    return acefa.load_library()


def _t(gtype, ne, es, data=1 << 20, nb=None):
    t = acefa.Tensor()
    t.type = gtype
    t.ne[:] = list(ne) + [1] * (4 - len(ne))
    if nb is None:
        nb = [es]
        for n in t.ne[:3]:
            nb.append(nb[-1] * max(1, n))
    t.nb[:] = nb
    t.data = data
    return t


def _cache(D=128, n=200, H=2, B=3, base=1 << 24, **change):
    nb = -(-n // 64)
    parts = {"k": _t(acefa.GGML_I8, (D, n, H, B), 1, base), "v": _t(acefa.GGML_I8, (D, n, H, B), 1, base + (1 << 22)),
             "k_scale": _t(acefa.GGML_F32, (nb, H, B), 4, base + (2 << 22)),
             "v_scale": _t(acefa.GGML_F32, (nb, H, B), 4, base + (3 << 22))}
    parts.update(change)
    return acefa.Kv8CacheC(parts["k"], parts["v"], parts["k_scale"], parts["v_scale"])


R = ctypes.byref
NO_DEVICE = (acefa.OK, -6, -7)  # accepted: only the device is missing here (or present, on a GPU machine)


def _store(lib, cache=None, k=None, v=None, cu=P, pos=P):
    k = k if k is not None else _t(acefa.GGML_F32, (128, 0, 2), 4, 1 << 28)
    v = v if v is not None else _t(acefa.GGML_F32, (128, 0, 2), 4, 1 << 29)
    return lib.acefa_kv8_store(R(cache or _cache()), R(k), R(v), cu, pos, None)


def test_store_refusals(lib):
    # (no rows: accepted calls launch nothing, so they are safe with addresses that are none)
    assert _store(lib) in NO_DEVICE
    assert _store(lib, pos=None) == -1
    assert lib.acefa_kv8_store(None, R(_t(0, (128, 0, 2), 4)), R(_t(0, (128, 0, 2), 4)), P, P, None) == -1
    f32 = acefa.GGML_F32
    assert _store(lib, k=_t(acefa.GGML_I8, (128, 6, 2), 1, 1 << 28), v=_t(acefa.GGML_I8, (128, 6, 2), 1, 1 << 29)) == -2
    assert _store(lib, k=_t(f32, (128, 6, 2), 4, 1 << 28), v=_t(acefa.GGML_F16, (128, 6, 2), 2, 1 << 29)) == -2
    bad = [((64, 6, 2), (64, 6, 2)), ((128, 6, 1), (128, 6, 1)), ((128, 6, 2), (128, 5, 2)), ((128, 6, 2, 2),) * 2]
    for a, b in bad:
        assert _store(lib, k=_t(f32, a, 4, 1 << 28), v=_t(f32, b, 4, 1 << 29)) == -3
    seven = [_t(f32, (128, 7, 2), 4, x) for x in (1 << 28, 1 << 29)]
    assert _store(lib, k=seven[0], v=seven[1], cu=None) == -3          # not a multiple of the sets
    assert _store(lib, k=_t(f32, (128, 6, 2), 4, 1 << 28, nb=[8, 1024, 8192, 8192])) == -4
    inside = _t(f32, (128, 6, 2), 4, (1 << 24) + 4096)
    assert _store(lib, k=inside, v=_t(f32, (128, 6, 2), 4, 1 << 29)) == -4  # overlaps the cache


def test_keys_and_values_of_one_buffer_are_accepted(lib):
    """k and v interleaved per set, per head or per row are no overlap; shifted by less than a row they are."""
    sets = [1, 128, 128 * 200, 2 * 2 * 128 * 200]
    heads = [1, 128, 2 * 128 * 200, 2 * 2 * 128 * 200]
    rows = [1, 256, 256 * 200, 2 * 256 * 200]
    for nb, step in ((sets, 2 * 128 * 200), (heads, 128 * 200), (rows, 128)):
        k, v = (_t(acefa.GGML_I8, (128, 200, 2, 3), 1, x, nb=nb) for x in (1 << 24, (1 << 24) + step))
        assert _store(lib, cache=_cache(k=k, v=v)) in NO_DEVICE
        v = _t(acefa.GGML_I8, (128, 200, 2, 3), 1, (1 << 24) + step - 16, nb=nb)
        assert _store(lib, cache=_cache(k=k, v=v)) == -4


@pytest.mark.parametrize("change,want", [
    ({"D": 96}, -3), ({"D": 256}, -3), ({"B": 1025}, -3), ({"H": 5000}, -3), ({"n": 0}, -3),
    ({"k": _t(acefa.GGML_F16, (128, 200, 2, 3), 2, 1 << 24)}, -2),
    ({"v": _t(acefa.GGML_I8, (128, 199, 2, 3), 1, 1 << 25)}, -3),
    ({"k_scale": _t(acefa.GGML_F32, (3, 2, 3), 4, 1 << 26)}, -3),
    ({"k_scale": _t(acefa.GGML_F16, (4, 2, 3), 2, 1 << 26)}, -2),
    ({"k": _t(acefa.GGML_I8, (128, 200, 2, 3), 1, (1 << 24) + 8)}, -4),
    ({"k": _t(acefa.GGML_I8, (128, 200, 2, 3), 1, 1 << 24, nb=[1, 136, 27200, 54400])}, -4),
    ({"k": _t(acefa.GGML_I8, (128, 200, 2, 3), 1, 1 << 24, nb=[1, 128, 25600, 0])}, -4),       # sets on one another
    ({"v": _t(acefa.GGML_I8, (128, 200, 2, 3), 1, 1 << 24)}, -4),                             # K on V
    ({"k": _t(acefa.GGML_I8, (128, 200, 2, 3), 1, 0)}, -1),
])
def test_cache_refusals(lib, change, want):
    assert _store(lib, cache=_cache(**change)) == want


def test_load_refusals(lib):
    f16 = acefa.GGML_F16

    def load(k, v, ln=P, cache=None):
        return lib.acefa_kv8_load(R(cache or _cache()), ln, R(k), R(v), None)

    ok = [_t(f16, (128, 100, 2, 3), 2, x) for x in (1 << 28, 1 << 29)]
    assert load(*ok, ln=None) == -1
    assert load(ok[0], _t(acefa.GGML_F32, (128, 100, 2, 3), 4, 1 << 29)) == -2
    assert load(*[_t(f16, (128, 201, 2, 3), 2, x) for x in (1 << 28, 1 << 29)]) == -3
    assert load(*[_t(f16, (128, 100, 2, 2), 2, x) for x in (1 << 28, 1 << 29)]) == -3
    assert load(ok[0], ok[0]) == -4
    assert load(_t(f16, (128, 100, 2, 3), 2, 1 << 24), ok[1]) == -4
    assert load(_t(f16, (128, 100, 2, 3), 2, 1 << 28, nb=[2, 128, 25600, 51200]), ok[1]) == -4  # rows overlap


def test_attend_refusals(lib):
    f32 = acefa.GGML_F32

    def attend(q=None, dst=None, weight=None, ln=P, scale=0.1, cache=None, ws=P, n=1 << 30):
        q = q if q is not None else _t(f32, (128, 1, 4, 3), 4, 1 << 28)
        dst = dst if dst is not None else _t(f32, (128, q.ne[2], q.ne[1], 3), 4, 1 << 29)
        return lib.acefa_kv8_attn(R(q), R(cache or _cache()), ln, R(dst), scale, R(weight) if weight else None, None,
                                  ws, n)

    assert attend(ln=None) == -1
    assert attend(q=_t(acefa.GGML_I8, (128, 1, 4, 3), 1, 1 << 28)) == -2
    assert attend(dst=_t(acefa.GGML_I8, (128, 4, 1, 3), 1, 1 << 29)) == -2
    for ne in ((64, 1, 4, 3), (128, 0, 4, 3), (128, 1, 3, 3), (128, 1, 4, 2), (128, 33, 4, 3), (128, 1, 130, 3)):
        assert attend(q=_t(f32, ne, 4, 1 << 28)) == -3, ne
    assert attend(dst=_t(f32, (128, 1, 4, 3), 4, 1 << 29)) == -3
    assert attend(scale=float("nan")) == -3 and attend(scale=float("inf")) == -3
    assert attend(weight=_t(f32, (199, 2, 3), 4, 1 << 27)) == -3
    assert attend(weight=_t(acefa.GGML_F16, (200, 2, 3), 2, 1 << 27)) == -2
    assert attend(weight=_t(f32, (200, 2, 3), 4, 1 << 27, nb=[4, 800, 0, 0])) == -4
    assert attend(weight=_t(f32, (200, 2, 3), 4, 1 << 28)) == -4     # on Q
    assert attend(dst=_t(f32, (128, 4, 1, 3), 4, 1 << 28)) == -4     # on Q
    assert attend(dst=_t(f32, (128, 4, 1, 3), 4, 1 << 24)) == -4     # on the cache
    assert attend(dst=_t(f32, (128, 4, 1, 3), 4, 1 << 29, nb=[4, 0, 2048, 2048])) == -4
    assert attend(q=_t(f32, (128, 1, 4, 3), 4, 1 << 28, nb=[8, 1024, 1024, 4096])) == -4
    q = _t(f32, (128, 1, 3, 3), 4, 1 << 28)
    assert lib.acefa_kv8_attn_workspace_bytes(R(q), R(_cache()), None) == 0


def test_evict_refusals(lib):
    f32, i32 = acefa.GGML_F32, acefa.GGML_I32
    out = dict(n=100, base=1 << 30)

    def evict(cache=None, weight=None, ln=P, first=4, recent=10, dst=None, kept=None, wo=None,
              lo=ctypes.c_void_p(1 << 12)):
        return lib.acefa_kv8_evict(R(cache or _cache()), R(weight or _t(f32, (200, 2, 3), 4, 1 << 27)), ln, first,
                                   recent, R(dst or _cache(**out)), R(kept or _t(i32, (100, 2, 3), 4, 1 << 28)),
                                   R(wo) if wo else None, lo, None)

    assert evict(ln=None) == -1 and evict(lo=None) == -1
    assert evict(weight=_t(i32, (200, 2, 3), 4, 1 << 27)) == -2
    assert evict(kept=_t(f32, (100, 2, 3), 4, 1 << 28)) == -2
    assert evict(weight=_t(f32, (100, 2, 3), 4, 1 << 27)) == -3
    assert evict(kept=_t(i32, (101, 2, 3), 4, 1 << 28)) == -3      # more than the smaller cache holds
    assert evict(kept=_t(i32, (0, 2, 3), 4, 1 << 28)) == -3
    assert evict(first=60, recent=41) == -3 and evict(first=-1) == -3 and evict(recent=-1) == -3
    assert evict(first=2 ** 62, recent=2 ** 62) == -3
    assert evict(dst=_cache(n=100, H=1, base=1 << 30)) == -3
    assert evict(dst=_cache(n=100, D=64, base=1 << 30)) == -3
    assert evict(dst=_cache(n=100)) == -4                          # on the cache
    assert evict(wo=_t(f32, (100, 2, 3), 4, 1 << 28)) == -4        # on kept
    assert evict(wo=_t(f32, (100, 2, 3), 4, 1 << 27)) == -4        # on the weights
    assert evict(ln=P, lo=ctypes.c_void_p(260)) == -4              # len_out on len


def test_packed_refusals(lib):
    f16, bf16, f32 = acefa.GGML_F16, acefa.GGML_BF16, acefa.GGML_F32

    def packed(q=None, k=None, v=None, dst=None, cu=P, cu_k=None, n=2, mask=0, window=0, scale=0.1):
        q = q if q is not None else _t(f16, (128, 0, 4), 2, 1 << 26)
        k = k if k is not None else _t(f16, (128, 50, 2), 2, 1 << 27)
        v = v if v is not None else _t(f16, (128, 50, 2), 2, 1 << 28)
        dst = dst if dst is not None else _t(f16, (128, 4, q.ne[1]), 2, 1 << 29)
        return lib.acefa_flash_attn_packed(R(q), R(k), R(v), R(dst), cu, cu_k, n, mask, window, scale, None)

    assert packed() in NO_DEVICE  # no rows: nothing would be launched
    assert packed(cu=None) == -1
    assert packed(q=_t(f16, (128, 5, 4), 2, 0)) == -1
    assert packed(q=_t(f32, (128, 0, 4), 4, 1 << 26)) == -2
    assert packed(k=_t(bf16, (128, 50, 2), 2, 1 << 27)) == -2
    assert packed(dst=_t(bf16, (128, 4, 0), 2, 1 << 29)) == -2
    assert packed(k=_t(f16, (128, 50, 3), 2, 1 << 27), v=_t(f16, (128, 50, 3), 2, 1 << 28)) == -3
    assert packed(v=_t(f16, (128, 49, 2), 2, 1 << 28)) == -3
    assert packed(q=_t(f16, (96, 0, 4), 2, 1 << 26)) == -3
    assert packed(dst=_t(f16, (128, 4, 1), 2, 1 << 29)) == -3
    assert packed(n=-1) == -3 and packed(n=70000) == -3 and packed(mask=3) == -3
    assert packed(mask=2, window=-1) == -3 and packed(scale=float("inf")) == -3
    assert packed(scale=0.0) == -3 and packed(scale=-0.1) == -3
    assert packed(q=_t(f16, (128, (1 << 24) + 1, 4), 2, 1 << 26)) == -3
    assert packed(k=_t(f16, (128, 50, 2), 2, (1 << 27) + 2)) == -4
    assert packed(k=_t(f16, (128, 50, 2), 2, 1 << 27, nb=[2, 264, 13200, 13200])) == -4
    assert packed(q=_t(f16, (128, 1, 4), 2, 1 << 26), dst=_t(f16, (128, 4, 1), 2, (1 << 29) + 1)) == -4
    assert packed(cu=ctypes.c_void_p(257)) == -4
    assert packed(k=_t(f16, (128, 50, 2), 2, 1 << 27, nb=[2, 256, 0, 0])) == -4
    q = _t(f16, (128, 7, 4), 2, 1 << 26)
    for nb in ([2, 256, 512, 0], [2, 128, 1024, 0], [2, 0, 256, 0], [2, 1024, 512, 0]):
        assert packed(q=q, dst=_t(f16, (128, 4, 7), 2, 1 << 29, nb=nb)) == -4, nb


def test_python_refusals():
    i8, f = torch.zeros((1, 1, 64, 64), dtype=torch.int8), torch.zeros((1, 1, 1))
    with pytest.raises(ValueError):
        acefa.Kv8Cache(i8.float(), i8, f, f)
    with pytest.raises(ValueError):
        acefa.Kv8Cache(i8, i8, f[0], f)
    cache = acefa.Kv8Cache(i8, i8.clone(), f, f.clone())
    x, pos = torch.zeros((1, 1, 64)), torch.zeros(1, dtype=torch.int32)
    for bad in (pos.long(), torch.zeros(2, dtype=torch.int32), pos[None]):
        with pytest.raises(ValueError):
            acefa.Kv8Store(cache, x, x, bad)
    with pytest.raises(acefa.AcefaError):
        acefa.Kv8Load(cache, pos, x[None].half(), x[None])()


def test_cache_structure_matches_the_header(tmp_path):
    import shutil
    import subprocess
    import os

    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "acefa.h"\nint main(void) { printf("%zu %zu %zu %zu", '
                   "sizeof(acefa_kv8_cache), offsetof(acefa_kv8_cache, v), offsetof(acefa_kv8_cache, k_scale), "
                   "offsetof(acefa_kv8_cache, v_scale)); return 0; }\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(root, "include"), str(src), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    C = acefa.Kv8CacheC
    assert got == [ctypes.sizeof(C), C.v.offset, C.k_scale.offset, C.v_scale.offset]
