"""A q4 projection of many tokens with a low-rank adapter per token
(osm_q4_project) against float64."""

import ctypes

import numpy as np
import pytest

import osm_hip
from helpers import bf16_bits, bf16_to_f32, pack_q4

pytestmark = pytest.mark.gpu

F32, F16, BF16 = osm_hip.F32, osm_hip.F16, osm_hip.BF16
U = 2.0**-24
HALF_STEP = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}


def stored(v, dtype):
    """(values in float64 as the device sees them, array to upload)."""
    v = np.ascontiguousarray(v, np.float32)
    if dtype == F32:
        return v.astype(np.float64), v
    if dtype == F16:
        h = v.astype(np.float16)
        return h.astype(np.float64), h
    b = bf16_bits(v).reshape(v.shape)
    return bf16_to_f32(b).astype(np.float64), b


class Problem:
    def __init__(self, ctx, T, N, K, group, meta=BF16, x=F32, y=None, count=0, rank=0, adapter=BF16, ragged=False, ids=None,
                 scales=True, x_pad=0, y_pad=0, seed=0, shift=0, on_device=True):
        rng = np.random.default_rng(seed + T * 7 + N * 3 + K)
        self.ctx, self.T, self.N, self.K, self.xt, self.yt = ctx, T, N, K, x, x if y is None else y
        self.x_stride, self.y_stride, self.group = K + x_pad, N + y_pad, group
        q = rng.integers(0, 16, (N, K), dtype=np.uint32)
        s = np.abs(rng.normal(0, 0.02, (N, K // group)))
        s64, self.s = stored(s, meta)
        b64, self.b = stored(-8 * s + rng.normal(0, 0.002, s.shape), meta)
        sq, bb = np.repeat(s64, group, 1) * q, np.repeat(b64, group, 1)
        self.packed = pack_q4(q)
        self.x64, xr = stored(rng.normal(size=(T, K)), x)
        rows = np.full((T + 1, self.x_stride), np.float32(7).astype(xr.dtype) if xr.dtype != np.uint16 else 0x40E0, xr.dtype)
        rows[:T, :K] = xr
        self.xd = self.upload(rows, shift * xr.itemsize)
        self.y_bytes = (T + 1) * self.y_stride * (4 if self.yt == F32 else 2)
        self.yd = ctx.alloc(self.y_bytes)
        if on_device:
            self.arrays = [self.upload(a) for a in (self.packed, self.s, self.b)]
            self.w = osm_hip.Q4ProjectionWeights.on_device(ctx, self.arrays[0].ptr, N, K // 8, self.arrays[1].ptr,
                                                           self.arrays[2].ptr, group, meta)
        else:
            self.w = osm_hip.Q4ProjectionWeights(ctx, self.packed, N, K // 8, self.s, self.b, group, meta)
        self.w64 = sq + bb
        self.y64 = self.x64 @ self.w64.T
        # No product meets more roundings than: the 66 of a matrix instruction's sum at each 32 columns of its chain, two for
        # each group's scale and bias, and 64 for the chains' sums. The activations may be held as two 11-bit terms (2^-22),
        # and what is far below a row's largest value in steps of 2^-38 of it.
        n = 66 * (K / 32) + 2 * (K / group) + 64
        mag = np.abs(self.x64) @ (np.abs(sq) + np.abs(bb)).T
        top = np.abs(self.x64).max(1, initial=0)[:, None] * (np.abs(sq) + np.abs(bb)).sum(1)[None]
        self.tol = (n * U + 2.0**-22) * mag + 2.0**-38 * top
        self.ad, self.ids = None, None
        if count:
            a64, ar = stored(rng.normal(size=(count, rank, K)) / np.sqrt(K), adapter)
            c64, br = stored(0.5 * rng.normal(size=(count, N, rank)), adapter)
            f = (0.5 + rng.random(count)).astype(np.float32)
            ranks = rng.integers(0 if count > 2 else 1, rank + 2, count).astype(np.uint32) if ragged else np.full(count, rank, np.uint32)
            if ragged:  # what lies beyond an adapter's rank is not used
                for i in range(count):
                    nan = np.uint16(0x7FC0) if adapter == BF16 else np.nan
                    ar[i, min(ranks[i], rank):] = nan
                    br[i, :, min(ranks[i], rank):] = nan
            self.ids = np.asarray(rng.integers(-1, count, T) if ids is None else ids, np.int32)
            self.dev = [self.upload(v) for v in (ar, br, f, ranks, self.ids)]
            self.ad = osm_hip.Adapters(self.dev[0].ptr, self.dev[1].ptr, count, rank, adapter,
                                       scales=self.dev[2].ptr if scales else None, ranks=self.dev[3].ptr if ragged else None)
            for t, i in enumerate(self.ids):
                if 0 <= i < count:
                    r, k = min(ranks[i], rank), float(f[i]) if scales else 1.0
                    v, vm = k * (a64[i, :r] @ self.x64[t]), abs(k) * (np.abs(a64[i, :r]) @ np.abs(self.x64[t]))
                    self.y64[t] += c64[i, :, :r] @ v
                    # Two chains and their splits into terms of 8 bits or more, three of them (two where y has 16 bits).
                    e = (66 * (K / 32) + 64 + 66 * (rank / 16 + 1) + 16) * U + (0 if self.yt == F32 else 2.0**-15)
                    self.tol[t] += e * (np.abs(c64[i, :, :r]) @ vm)
        self.tol = self.tol + HALF_STEP[self.yt] * (np.abs(self.y64) + self.tol) + (2.0**-25 if self.yt == F16 else 0)

    def upload(self, a, shift=0):
        d = self.ctx.alloc(a.nbytes + 64)
        d.upload(np.concatenate([np.zeros(shift, np.uint8), np.ascontiguousarray(a).view(np.uint8).reshape(-1)]))
        if shift:
            d.ptr = ctypes.c_void_p(d.ptr.value)
            d.at = ctypes.c_void_p(d.ptr.value + shift)
        else:
            d.at = d.ptr
        return d

    def call(self):
        osm_hip.q4_project(self.ctx, self.w, self.xd.at, self.yd.ptr, self.T, x_dtype=self.xt, y_dtype=self.yt,
                           x_stride=self.x_stride, y_stride=self.y_stride, adapters=self.ad,
                           adapter_ids_ptr=self.dev[4].ptr if self.ad is not None else None)

    def run(self):
        fill = np.full(self.y_bytes, 0xAB, np.uint8)
        self.yd.upload(fill)
        self.call()
        raw = self.yd.download(np.uint8, self.y_bytes)
        y = raw.view({F32: np.float32, F16: np.float16, BF16: np.uint16}[self.yt]).reshape(self.T + 1, self.y_stride)
        used = np.zeros(y.shape, bool)
        used[:self.T, :self.N] = True
        assert np.all(raw.reshape(self.T + 1, self.y_stride, -1)[~used] == 0xAB)  # between rows and behind them: as it was
        got = y[:self.T, :self.N]
        return bf16_to_f32(got) if self.yt == BF16 else got

    def check(self):
        y = self.run().astype(np.float64)
        over = np.abs(y - self.y64) / self.tol
        assert np.all(over <= 1), float(over.max())


# tokens: one, fewer than a tile, tiles and one more, a long run; rows and columns that fill no tile; groups of any size.
@pytest.mark.parametrize("T,N,K,group", [
    (1, 1, 32, 32), (1, 512, 512, 64), (2, 130, 1024, 128), (5, 67, 96, 32), (16, 64, 256, 64), (17, 65, 320, 64),
    (33, 200, 2048, 64), (64, 257, 640, 128), (65, 31, 512, 32), (129, 384, 512, 64), (300, 129, 1056, 32), (520, 1000, 256, 64),
    (3, 40, 96, 96), (70, 50, 8, 8), (9, 33, 40, 40), (20, 19, 72, 24), (66, 140, 192, 48), (130, 20, 56, 7)])
@pytest.mark.parametrize("x", [F32, F16, BF16])
def test_matches_float64(ctx, T, N, K, group, x):
    print(f"[project] T={T} N={N} K={K} group={group} x={x}", flush=True)
    meta = (F32, F16, BF16)[(T + x) % 3]
    adapter = (F32, F16, BF16)[(N + 2 * x) % 3]
    Problem(ctx, T, N, K, group, meta, x).check()
    Problem(ctx, T, N, K, group, meta, x, y=F32, count=5, rank=16, adapter=adapter).check()


# Enough tokens and rows for the larger tiles, whole and ragged, over few columns.
@pytest.mark.parametrize("T,N,K,group", [(1000, 4090, 160, 32), (1024, 4096, 320, 64), (2040, 4095, 96, 32), (2048, 4096, 448, 64)])
@pytest.mark.parametrize("x", [F32, F16, BF16])
def test_large_tiles(ctx, T, N, K, group, x):
    print(f"[project] T={T} N={N} K={K} group={group} x={x}", flush=True)
    for meta in (F32, F16, BF16):
        Problem(ctx, T, N, K, group, meta, x, count=5 if meta == BF16 else 0, rank=24, ragged=True, y_pad=8 * (meta == F16)).check()


# fp32 in and out: the outputs' rms error is at most that of one fp32 sum over the columns in turn. Each of its K roundings is
# 2^-25 rms of a partial sum, which grows as the square root of its terms: together 2^-25 sqrt(K / 2) of the result.
@pytest.mark.parametrize("T,N", [(1, 512), (12, 256), (37, 256), (64, 8192), (100, 256), (2048, 4096)])
@pytest.mark.parametrize("K,group", [(2048, 32), (4096, 64), (4096, 128)])
def test_sums_are_fp32(ctx, T, N, K, group):
    print(f"[project] T={T} N={N} K={K} group={group}", flush=True)
    for x in (F32, F16, BF16):
        for count in (0, 4):
            p = Problem(ctx, T, N, K, group, F32, x, y=F32, count=count, rank=16, adapter=F32)
            off = p.run() - p.y64
            assert np.sqrt(np.mean(off**2) / np.mean(p.y64**2)) <= 2.0**-25 * np.sqrt(K / 2)


def test_as_many_tokens_as_a_call_takes(ctx):
    T = 1 << 20
    ids = np.full(T, -1)
    ids[[0, 1, 70001, T - 2, T - 1]] = 0, 1, 1, 1, 0
    for N, K, group, rank in ((1, 8, 8, 64), (32, 32, 32, 8)):
        print(f"[project] T={T} N={N} K={K} group={group}", flush=True)
        Problem(ctx, T, N, K, group, BF16, BF16, count=2, rank=rank, ids=ids).check()


def test_more_adapters_than_are_sorted(ctx):
    for x in (F32, BF16):
        for T in (3, 30, 130):
            ids = np.arange(T) * 521 % 65537
            ids[0], ids[T - 1], ids[1] = 65536, 65537, 65536
            Problem(ctx, T, 40, 32, 32, BF16, x, count=65537, rank=1, ids=ids).check()


@pytest.mark.parametrize("rank", [1, 3, 8, 16, 21, 64, 130, 256])
@pytest.mark.parametrize("adapter", [F32, F16, BF16])
@pytest.mark.parametrize("T", [1, 40, 200])
def test_ranks_and_types(ctx, rank, adapter, T):
    print(f"[project] rank={rank} adapter={adapter} T={T}", flush=True)
    for x, ragged, scales in ((F32, False, True), (F16, True, False), (BF16, True, True)):
        Problem(ctx, T, 300, 512, 64, BF16, x, count=7, rank=rank, adapter=adapter, ragged=ragged, scales=scales).check()


@pytest.mark.parametrize("ids", ["none", "outside", "one", "each", "runs", "two"])
@pytest.mark.parametrize("T", [1, 30, 64, 150, 700])
def test_adapter_ids(ctx, ids, T):
    count = 64
    i = np.arange(T)
    picked = {"none": np.full(T, -1), "outside": np.where(i % 3 == 0, i % count, np.where(i % 3 == 1, count, -(2**31))),
              "one": np.full(T, 63), "each": i % count, "runs": i * 5 // T, "two": np.where(i == T // 2, 7, 3)}[ids]
    print(f"[project] ids={ids} T={T}", flush=True)
    for x in (F32, BF16):
        Problem(ctx, T, 210, 256, 64, F32, x, count=count, rank=8, ids=picked).check()


@pytest.mark.parametrize("x,y", [(F32, BF16), (F32, F16), (BF16, F32), (F16, F32), (BF16, F16), (F16, BF16)])
@pytest.mark.parametrize("T", [1, 50, 260])
def test_types_strides_and_alignment(ctx, x, y, T):
    for pad, shift in ((0, 1), (1, 0), (8, 0), (13, 3)):
        print(f"[project] x={x} y={y} T={T} pad={pad} shift={shift}", flush=True)
        Problem(ctx, T, 193, 512, 64, BF16, x, y=y, count=3, rank=12, x_pad=pad, y_pad=pad, shift=shift).check()
    Problem(ctx, T, 193, 512, 64, BF16, x, y=y, on_device=False).check()


def test_values_of_every_size(ctx):
    # Rows of very different scale, rows with values far below their largest, a row of zeros.
    for x in (F32, BF16):
        for T in (9, 150):
            p = Problem(ctx, T, 96, 512, 64, F32, x)
            scale = np.ones((T, 512))
            scale[0], scale[1], scale[2, 1:], scale[3], scale[4, ::2] = 1e30, 1e-30, 2.0**-20, 0.0, 2.0**-9
            p.x64, xr = stored((p.x64 * scale).astype(np.float32), x)
            p.xd = p.upload(xr)
            y64 = p.x64 @ p.w64.T
            mag = np.abs(p.x64) @ np.abs(p.w64).T * 17 + np.abs(p.x64).max(1)[:, None] * 512 * 2.0**-16  # |s q| + |b| <= 17 |w| on the whole
            bound = mag * (2.0**-22 + 2000 * U) + HALF_STEP[x] * np.abs(y64) + 1e-37
            y = p.run().astype(np.float64)
            assert np.all(np.isfinite(y)) and np.all(np.abs(y - y64) <= bound)


def test_a_row_that_is_not_finite_stays_alone(ctx):
    for x in (F32, F16, BF16):
        for T in (4, 150):
            p = Problem(ctx, T, 140, 512, 64, BF16, x, count=4, rank=8, ids=np.arange(T) % 4)
            ref = p.run().copy()
            bad = p.x64.astype(np.float32)
            bad[1, 5], bad[2, 7] = np.nan, np.inf
            p.xd = p.upload(stored(np.where(np.isfinite(bad), bad, 0), x)[1])
            raw = stored(np.where(np.isfinite(bad), bad, 0), x)[1]
            raw[1, 5], raw[2, 7] = {F32: (np.nan, np.inf), F16: (np.nan, np.inf), BF16: (0x7FC0, 0x7F80)}[x]
            p.xd = p.upload(raw)
            got = p.run()
            rest = np.ones(T, bool)
            rest[1:3] = False
            assert np.array_equal(got[rest], ref[rest])
            # An adapter that is not finite reaches its own tokens only.
            p = Problem(ctx, T, 140, 512, 64, BF16, x, count=4, rank=8, ids=np.arange(T) % 4)
            ref = p.run().copy()
            nan = np.full(140 * 8, 0x7FC0, np.uint16)
            host = p.dev[1].download(np.uint16, 4 * 140 * 8)
            host[:140 * 8] = nan
            p.dev[1].upload(host)
            got = p.run()
            assert np.array_equal(got[np.arange(T) % 4 != 0], ref[np.arange(T) % 4 != 0])
            assert np.all(np.isnan(got[0]))


def test_repeats_graphs_and_two_contexts(ctx):
    a = Problem(ctx, 150, 260, 512, 64, BF16, BF16, count=6, rank=16)
    b = Problem(ctx, 7, 260, 512, 64, BF16, F32, count=6, rank=16)
    big = Problem(ctx, 600, 260, 1024, 64, BF16, F32, count=6, rank=64)
    ra, rb = a.run().copy(), b.run().copy()
    big.run()  # the workspace as large as it gets here
    with ctx.capture() as one:
        a.call()
        b.call()
    with ctx.capture() as two:
        b.call()
        a.call()
    for g in (one, two, one, two):
        a.yd.upload(np.zeros(a.y_bytes, np.uint8))
        b.yd.upload(np.zeros(b.y_bytes, np.uint8))
        g.graph.launch()
        ctx.synchronize()
        for p, ref in ((a, ra), (b, rb)):
            raw = p.yd.download(np.uint8, p.y_bytes)
            y = raw.view(np.float32 if p.yt == F32 else np.uint16).reshape(p.T + 1, p.y_stride)[:p.T, :p.N]
            assert np.array_equal(bf16_to_f32(y) if p.yt == BF16 else y, ref)
        big.check()  # other work in the same workspace between the replays
    # Another context has a workspace and a stream of its own: calls of both at once.
    other = osm_hip.Context(0)
    c = Problem(other, 150, 260, 512, 64, BF16, BF16, count=6, rank=16)
    for _ in range(5):
        c.call()
        a.call()
        b.call()
    assert np.array_equal(c.run(), ra) and np.array_equal(a.run(), ra) and np.array_equal(b.run(), rb)
    del c
    other.close()


def test_workspace_does_not_grow_in_a_capture(ctx):
    fresh = osm_hip.Context(0)
    p = Problem(fresh, 64, 64, 512, 64, BF16, F32, count=2, rank=8)
    with fresh.capture() as cap:
        with pytest.raises(osm_hip.OsmError) as e:
            p.call()
        osm_hip.group_rows(fresh, p.dev[4].ptr, 8, 2, p.yd.ptr, p.yd.ptr.value + 64)
    assert "capture" in e.value.diagnostic
    cap.graph.launch()
    p.check()
    fresh.close()


def test_no_tokens(ctx):
    p = Problem(ctx, 3, 64, 512, 64)
    osm_hip.q4_project(ctx, p.w, None, None, 0)


def test_refused(ctx):
    p = Problem(ctx, 4, 64, 512, 64, count=2, rank=8)
    x, y, ids = p.xd.ptr, p.yd.ptr, p.dev[4].ptr
    odd = ctypes.c_void_p(x.value + 1)

    def adapters(**kw):
        d = dict(a_ptr=p.dev[0].ptr, b_ptr=p.dev[1].ptr, count=2, max_rank=8, dtype=BF16)
        return osm_hip.Adapters(**{**d, **kw})

    for kw in (dict(x_ptr=None), dict(y_ptr=None), dict(x_dtype=3), dict(y_dtype=7), dict(x_stride=511), dict(y_stride=63),
               dict(tokens=(1 << 20) + 1), dict(x_ptr=odd), dict(y_ptr=odd), dict(adapters=adapters(count=0)),
               dict(adapters=adapters(max_rank=0)), dict(adapters=adapters(max_rank=257)), dict(adapters=adapters(dtype=3)),
               dict(adapters=adapters(a_ptr=None)), dict(adapters=adapters(b_ptr=odd)), dict(adapter_ids_ptr=None),
               dict(adapters=adapters(scales=odd)), dict(adapters=adapters(count=2**32 - 1))):
        call = {**dict(x_ptr=x, y_ptr=y, tokens=4, adapters=adapters(), adapter_ids_ptr=ids), **kw}
        with pytest.raises(osm_hip.OsmError) as e:
            osm_hip.q4_project(ctx, p.w, **call)
        assert e.value.status == osm_hip.OSM_E_INVALID and e.value.diagnostic, kw
    a = [v.ptr for v in p.arrays]
    off = lambda v: ctypes.c_void_p(v.value + 4)  # noqa: E731
    for args in ((None, 64, 64, a[1], a[2], 64), (a[0], 0, 64, a[1], a[2], 64), (a[0], 64, 64, a[1], a[2], 48),
                 (a[0], 64, 64, a[1], a[2], 0), (off(a[0]), 64, 64, a[1], a[2], 64), (a[0], 64, 64, off(a[1]), a[2], 64),
                 (a[0], 64, 64, a[1], None, 64)):
        with pytest.raises(osm_hip.OsmError) as e:
            osm_hip.Q4ProjectionWeights.on_device(ctx, *args, meta_dtype=BF16)
        assert e.value.status == osm_hip.OSM_E_INVALID


def test_gemv_reads_arrays_on_the_device(ctx):
    p, q = Problem(ctx, 1, 320, 512, 64, BF16, F32), Problem(ctx, 1, 320, 512, 64, BF16, F32, on_device=False)
    xb, yb, zb = osm_hip.FloatBuffer(ctx, 512), osm_hip.FloatBuffer(ctx, 320), osm_hip.FloatBuffer(ctx, 320)
    xb.upload(p.x64.astype(np.float32).reshape(-1))
    osm_hip.run_q4_gemv_preloaded(ctx, p.w, xb, yb)
    osm_hip.run_q4_gemv_preloaded(ctx, q.w, xb, zb)
    assert np.array_equal(yb.download(), zb.download())
