"""CPU tests of the packed and 8-bit-cache entries at the edges of what they accept."""
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
