"""Rows grouped by key (osm_group_rows) against numpy's stable sort."""

import ctypes

import numpy as np
import pytest

import osm_hip

pytestmark = pytest.mark.gpu


def group(ctx, keys, buckets):
    n = keys.size
    k, off, order = ctx.alloc(4 * n + 64), ctx.alloc(4 * (buckets + 1) + 64), ctx.alloc(4 * n + 64)
    k.upload(np.concatenate([keys, np.zeros(16, np.int32)]))  # rows behind the last: key 0, not counted
    for a in (off, order):
        a.upload(np.full(a.nbytes // 4, 0xABABABAB, np.uint32))
    osm_hip.group_rows(ctx, k.ptr, n, buckets, off.ptr, order.ptr)
    ctx.synchronize()
    o, r = off.download(np.uint32, off.nbytes // 4), order.download(np.uint32, order.nbytes // 4)
    assert np.all(o[buckets + 1:] == 0xABABABAB) and np.all(r[n:] == 0xABABABAB)
    return o[:buckets + 1], r[:n]


def expected(keys, buckets):
    b = np.where((keys >= 0) & (keys < buckets), keys, buckets)
    counts = np.bincount(b, minlength=buckets + 1)
    return np.cumsum(counts) - counts, np.argsort(b, kind="stable")


@pytest.mark.parametrize("n", [0, 1, 63, 64, 65, 1000, 1025, 4097, 16384, 16385, 81920, 300007, 1100003])
@pytest.mark.parametrize("buckets", [1, 2, 7, 255, 256, 512, 1000, 2047, 2048, 65535])
def test_matches_stable_sort(ctx, n, buckets):
    rng = np.random.default_rng(n + buckets)
    print(f"[group] n={n} buckets={buckets}", flush=True)
    uniform = rng.integers(0, buckets, n)
    skewed = np.minimum(rng.geometric(0.3, n) - 1, buckets - 1)
    keys = {"uniform": uniform, "outside": np.where(rng.random(n) < 0.3, rng.choice([-1, buckets, -(2**31), 2**31 - 1], n), uniform),
            "skewed": skewed, "one": np.full(n, buckets - 1), "sorted": np.sort(uniform), "none": np.full(n, -5)}
    for name, k in keys.items():
        k = k.astype(np.int32)
        offsets, order = group(ctx, k, buckets)
        ref_offsets, ref_order = expected(k, buckets)
        assert np.array_equal(offsets, ref_offsets), name
        assert np.array_equal(order, ref_order), name


def test_many_rows_in_a_capture(ctx):
    # The counts of many rows are in the context's workspace: it does not grow while a capture is recording.
    rng = np.random.default_rng(3)
    fresh = osm_hip.Context(0)
    n, buckets = 50001, 300
    keys, offsets, order = fresh.alloc(4 * n), fresh.alloc(4 * (buckets + 1)), fresh.alloc(4 * n)
    with fresh.capture() as small:
        with pytest.raises(osm_hip.OsmError) as e:
            osm_hip.group_rows(fresh, keys.ptr, n, buckets, offsets.ptr, order.ptr)
        osm_hip.group_rows(fresh, keys.ptr, 9, 1, offsets.ptr, order.ptr)
    assert "capture" in e.value.diagnostic
    keys.upload(np.zeros(n, np.int32))
    small.graph.launch()
    osm_hip.group_rows(fresh, keys.ptr, n, buckets, offsets.ptr, order.ptr)
    with fresh.capture() as cap:
        osm_hip.group_rows(fresh, keys.ptr, n, buckets, offsets.ptr, order.ptr)
    for _ in range(3):
        k = rng.integers(-1, buckets + 1, n).astype(np.int32)
        keys.upload(k)
        cap.graph.launch()
        fresh.synchronize()
        ref_offsets, ref_order = expected(k, buckets)
        assert np.array_equal(offsets.download(np.uint32, buckets + 1), ref_offsets)
        assert np.array_equal(order.download(np.uint32, n), ref_order)
        assert np.array_equal(group(fresh, k[::-1].copy(), 7)[1], expected(k[::-1], 7)[1])  # other work in the same workspace
    fresh.close()


def test_refused(ctx):
    a = ctx.alloc(256)
    odd = ctypes.c_void_p(a.ptr.value + 2)
    for args in ((a.ptr, 4, 0, a.ptr, a.ptr), (a.ptr, 4, 65536, a.ptr, a.ptr), (None, 4, 2, a.ptr, a.ptr), (a.ptr, 4, 2, None, a.ptr),
                 (a.ptr, 4, 2, a.ptr, None), (odd, 4, 2, a.ptr, a.ptr), (a.ptr, 2**31, 2, a.ptr, a.ptr)):
        with pytest.raises(osm_hip.OsmError) as e:
            osm_hip.group_rows(ctx, *args)
        assert e.value.status == osm_hip.OSM_E_INVALID and e.value.diagnostic
