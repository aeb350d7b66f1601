"""The 4-bit storage mode without a device: pools, sizes and refusals."""
import pytest

import krill_amd
from krill_amd import _lib as L
from krill_amd._lib import KrillError


def test_host_only_pool_counts_half_bytes():
    for D in (64, 128, 256, 512):
        pool = krill_amd.KVPool(2, 3, D, 8, "affine4_g64", "bf16", host_only=True)
        s = pool.seq_create()
        pool.reserve_append(s, 100)
        per_token = 3 * (D + 8 * (D // 64))
        assert pool.seq_memory_bytes(s) == 100 * per_token
        assert pool.stats()["block_bytes"] == 64 * per_token
        pool.close()


def test_kernels_need_device_memory():
    pool = krill_amd.KVPool(1, 1, 64, 4, "affine4_g64", "f16", host_only=True)
    for call in ("krill_read_slots", "krill_gather", "krill_scatter"):
        args = {"krill_read_slots": (pool.handle, 0, None, 1, 1, None, None, None),
                "krill_gather": (pool.handle, 0, None, None, 1, 1, 1, 0, None, None),
                "krill_scatter": (pool.handle, 0, None, 1, 1, None, None, 1, None)}[call]
        assert getattr(L.lib(), call)(*args) == L.KRILL_E_STATE
    pool.close()


def test_unknown_mode_is_refused():
    desc = L.PoolDesc(1, 1, 64, 64, 4, 3, L.DTYPE_BF16, L.POOL_HOST_ONLY, 0.0, 0, 0, -1, 0)
    import ctypes

    h = ctypes.c_void_p()
    assert L.lib().krill_pool_create(ctypes.byref(desc), None, ctypes.byref(h)) == L.KRILL_E_INVAL
    with pytest.raises(KeyError):
        krill_amd.KVPool(1, 1, 64, 4, "affine3_g64", host_only=True)


@pytest.mark.parametrize("Hq,Lq", [(4, 1), (4, 8), (40, 1), (4, 512)])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_workspace_covers_every_call(D, Hq, Lq):
    pool = krill_amd.KVPool(1, 2, D, 4, "affine4_g64", host_only=True)
    assert pool.workspace_size(3, Hq, Lq, 1000) > 0
    with pytest.raises(KrillError) as e:
        pool.workspace_size(3, 3, Lq, 1000)
    assert e.value.code == L.KRILL_E_INVAL
    pool.close()


def test_prefix_cache_has_no_disk_tier(tmp_path):
    from krill_amd.cache import PrefixCache

    pool = krill_amd.KVPool(1, 1, 64, 4, "affine4_g64", host_only=True)
    with pytest.raises(ValueError):
        PrefixCache(pool, cache_dir=str(tmp_path))
    pc = PrefixCache(pool)
    assert pc._entry_bytes(10) == 10 * (64 + 8)
    pool.close()
