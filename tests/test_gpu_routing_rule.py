"""Routing to experts by a rule: osm_route_experts against its definition in
float64, and layers that route by one (osm_moe_layer_set_routing) on every
path."""

import ctypes

import numpy as np
import pytest

import oracle as O
import osm_hip
from helpers import bf16_bits, bf16_to_f32, rel_l2
from rule_reference import route

pytestmark = pytest.mark.gpu

SOFTMAX, SIGMOID = osm_hip.SCORE_SOFTMAX, osm_hip.SCORE_SIGMOID
# Scores and weights are formed in fp64 and rounded once: half a step of fp32, and what fp64's own exp, sum and divide add.
REL = 2.0**-24 + 1e-13


def stored(values, dtype):
    """(values as the device sees them, array to upload)."""
    v = values.astype(np.float32)
    if dtype == osm_hip.F32:
        return v, v
    if dtype == osm_hip.F16:
        h = v.astype(np.float16)
        return h.astype(np.float32), h
    with np.errstate(invalid="ignore"):
        b = np.where(np.isfinite(v), bf16_bits(np.where(np.isfinite(v), v, 0)), (v.view(np.uint32) >> 16).astype(np.uint16))
    return bf16_to_f32(b), b


def run(ctx, rule, logits, dtype, bias=None, stride=None, mass=True):
    T, E = logits.shape
    stride = stride or E
    seen, raw = stored(logits, dtype)
    rows = np.full((T, stride), 77, raw.dtype)  # what lies between rows is not read as a logit
    rows[:, :E] = raw
    k = rule.top_k
    lg, ids, w, m = ctx.alloc(max(rows.nbytes, 4)), ctx.alloc(4 * T * k + 64), ctx.alloc(4 * T * k + 64), ctx.alloc(4 * T + 64)
    lg.upload(rows)
    for a in (ids, w, m):
        a.upload(np.full(a.nbytes // 4, 0xABABABAB, np.uint32))
    b = None
    if bias is not None:
        b = ctx.alloc(4 * E)
        b.upload(bias.astype(np.float32))
    osm_hip.route_experts(ctx, rule, lg.ptr, dtype, T, ids.ptr, w.ptr, bias_ptr=b.ptr if b else None,
                          mass_ptr=m.ptr if mass else None, logits_stride=stride)
    ctx.synchronize()
    for a, n in ((ids, T * k), (w, T * k), (m, T if mass else 0)):
        assert np.all(a.download(np.uint32, a.nbytes // 4)[n:] == 0xABABABAB)
    return (seen, ids.download(np.uint32, T * k).reshape(T, k), w.download(np.float32, T * k).reshape(T, k),
            m.download(np.float32, T))


def check(ctx, rule, logits, dtype=osm_hip.F32, bias=None, stride=None):
    seen, ids, w, m = run(ctx, rule, logits, dtype, bias, stride)
    rid, rw, rm = route(seen, rule, bias)
    assert np.array_equal(ids, rid)
    assert np.all(np.abs(w - rw) <= REL * np.abs(rw) + 1e-45)
    assert np.all(np.abs(m - rm) <= REL * np.abs(rm) + 1e-45)


# E, k, score, groups, top_groups, group_score, bias: one expert, a whole wavefront and one more, sizes that fill no register
# run, every pick taken, groups of one expert, groups across lanes, the largest.
RULES = [
    (1, 1, SOFTMAX, 1, 1, 1, False), (7, 7, SIGMOID, 1, 1, 1, True), (8, 2, SOFTMAX, 1, 1, 1, False),
    (60, 6, SIGMOID, 4, 3, 2, True), (64, 64, SOFTMAX, 1, 1, 1, True), (64, 8, SIGMOID, 64, 8, 1, False),
    (65, 5, SIGMOID, 5, 2, 2, False), (128, 8, SOFTMAX, 8, 3, 1, True), (130, 10, SIGMOID, 1, 1, 1, True),
    (160, 6, SOFTMAX, 8, 3, 1, False), (256, 8, SIGMOID, 8, 4, 2, True), (384, 8, SIGMOID, 1, 1, 1, True),
    (512, 10, SOFTMAX, 1, 1, 1, False), (1000, 22, SIGMOID, 10, 4, 2, True), (1024, 16, SOFTMAX, 2, 1, 2, True),
]


@pytest.mark.parametrize("E,k,score,groups,top_groups,group_score,bias", RULES)
@pytest.mark.parametrize("dtype", [osm_hip.F32, osm_hip.F16, osm_hip.BF16])
def test_route_matches_definition(ctx, E, k, score, groups, top_groups, group_score, bias, dtype):
    rng = np.random.default_rng(E * 31 + k)
    b = (0.1 * rng.normal(size=E)).astype(np.float32) if bias else None
    for T, renorm, scale in ((1, True, 1.0), (67, False, 2.5), (130, True, 2.5)):
        print(f"[route] E={E} T={T}", flush=True)
        rule = osm_hip.RouteRule(E, k, score, groups, top_groups, group_score, renorm, scale)
        check(ctx, rule, 2 * rng.normal(size=(T, E)), dtype, b, stride=E + (0 if T == 67 else 3))


@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups", [1, 8])
def test_ties_masks_and_infinities(ctx, score, bias, groups):
    E, k = 256, 8
    rng = np.random.default_rng(5)
    x = np.round(2 * rng.normal(size=(40, E))) / 2  # few distinct logits: ties everywhere
    x[1] = 0.0                                      # all equal, of both signs of zero
    x[1, ::3] = -0.0
    x[2] = -np.inf                                  # nothing left
    x[3, 5:] = -np.inf                              # fewer than k left
    x[4] = np.nan
    x[5, rng.random(E) < 0.9] = -np.inf
    x[6, rng.random(E) < 0.3] = np.nan
    x[7] = np.finfo(np.float32).min
    x[8, rng.random(E) < 0.97] = np.finfo(np.float32).min
    x[9, [3, 200]] = np.inf
    x[10] = 80 + rng.normal(size=E)                 # sigmoids of 1
    x[11] = -90 + rng.normal(size=E)
    x[12] = np.linspace(-700, 700, E)
    x[13, 32:] = -np.inf                            # one whole group, the others empty
    b = (np.round(4 * rng.normal(size=E)) / 8).astype(np.float32) if bias else None
    if bias:
        b[[0, 77]] = -np.inf                        # experts taken out by the bias
        b[123] = np.inf                             # and one always in
    for renorm in (True, False):
        rule = osm_hip.RouteRule(E, k, score, groups, max(1, groups // 2), 2 if groups > 1 else 1, renorm, 1.0)
        check(ctx, rule, x, osm_hip.F32, b)


def test_next_to_the_border(ctx):
    # Choices that differ by less than a step of fp32: the sums rank in fp64.
    E = 128
    logits = np.zeros((3, E), np.float32)
    logits[:, :] = -3.0
    logits[0, 90], logits[0, 20] = np.nextafter(np.float32(2.0), np.float32(3)), 2.0
    logits[1, 90], logits[1, 20] = 2.0, np.nextafter(np.float32(2.0), np.float32(3))
    logits[2, 90], logits[2, 20] = 30.0, 29.99999  # sigmoids that round to one fp32 value
    bias = np.full(E, 0.125, np.float32)
    check(ctx, osm_hip.RouteRule(E, 1, SIGMOID), logits, bias=bias)
    check(ctx, osm_hip.RouteRule(E, 1, SOFTMAX), logits, bias=bias)


def test_no_tokens_and_repeats(ctx):
    rule = osm_hip.RouteRule(64, 4)
    osm_hip.route_experts(ctx, rule, None, osm_hip.F32, 0, None, None)
    rng = np.random.default_rng(2)
    x = rng.normal(size=(999, 64))
    first = run(ctx, rule, x, osm_hip.BF16)
    again = run(ctx, rule, x, osm_hip.BF16, mass=False)
    assert all(np.array_equal(a, b) for a, b in zip(first[:3], again[:3]))


@pytest.mark.parametrize("fields,why", [
    (dict(expert_count=0), "expert_count"), (dict(expert_count=1025), "expert_count"), (dict(top_k=0), "top_k"),
    (dict(top_k=65), "top_k"), (dict(groups=4, top_groups=1, top_k=17), "top_k"), (dict(score=2), "score"),
    (dict(groups=0), "groups"), (dict(groups=3), "groups"), (dict(groups=65), "groups"),
    (dict(groups=4, top_groups=5), "top_groups"), (dict(groups=4, top_groups=0), "top_groups"),
    (dict(group_score=0), "group_score"), (dict(group_score=3), "group_score"),
    (dict(groups=64, top_groups=64, group_score=2), "group_score"), (dict(scale=float("nan")), "scale")])
def test_refused_rules(ctx, fields, why):
    a = ctx.alloc(4096)
    rule = osm_hip.RouteRule(**{**dict(expert_count=64, top_k=4), **fields})
    with pytest.raises(osm_hip.OsmError) as e:
        osm_hip.route_experts(ctx, rule, a.ptr, osm_hip.F32, 1, a.ptr, a.ptr)
    assert e.value.status == osm_hip.OSM_E_INVALID and why in e.value.diagnostic


def test_refused_arguments(ctx):
    a = ctx.alloc(4096)
    rule = osm_hip.RouteRule(64, 4)
    call = lambda *v, **kw: osm_hip.route_experts(ctx, rule, *v, **kw)  # noqa: E731
    odd = ctypes.c_void_p(a.ptr.value + 1)
    for args, kw in (((None, 0, 1, a.ptr, a.ptr), {}), ((a.ptr, 0, 1, None, a.ptr), {}), ((a.ptr, 0, 1, a.ptr, None), {}),
                     ((a.ptr, 3, 1, a.ptr, a.ptr), {}), ((a.ptr, 0, 1, a.ptr, a.ptr), dict(logits_stride=63)),
                     ((a.ptr, 0, (1 << 20) + 1, a.ptr, a.ptr), {}), ((odd, 0, 1, a.ptr, a.ptr), {}),
                     ((a.ptr, 0, 1, a.ptr, a.ptr), dict(bias_ptr=odd))):
        with pytest.raises(osm_hip.OsmError) as e:
            call(*args, **kw)
        assert e.value.status == osm_hip.OSM_E_INVALID and e.value.diagnostic


# ---- layers that route by a rule ---------------------------------------------------------
SEED, D, I, G, E, K = 17, 512, 128, 64, 64, 6


@pytest.fixture(scope="module")
def model(ctx):
    g = osm_hip.geometry(D, I, G, osm_hip.BF16)
    slab = osm_hip.ExpertSlab(ctx, g, 1, E)
    slab.synthesize(SEED)
    store = osm_hip.ExpertStore(g, 1, E)
    store.synthesize(ctx, SEED)
    cache = osm_hip.ExpertCache(ctx, E * osm_hip.expert_blob_bytes(g), store=store)

    def layer(router=osm_hip.BF16, shared=True):
        w = O.synth_router_bf16(SEED, 0, E, D)
        sg = O.synth_shared_gate_bf16(SEED, 0, D)
        if router == osm_hip.F32:
            w, sg = bf16_to_f32(w), bf16_to_f32(sg)
        return osm_hip.MoeLayer(ctx, g, E, K, w, router, sg if shared else None, O.synth_norm_weight(SEED, 0, D),
                                O.synth_expert_blob(SEED, 0, O.SHARED_EXPERT_ID, D, I, G) if shared else None, max_tokens=256)

    return slab, store, cache, layer


RULE = dict(score=SIGMOID, groups=8, top_groups=3, group_score=2, renormalize=True, scale=2.5)


@pytest.mark.parametrize("router", [osm_hip.BF16, osm_hip.F32])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("path", [osm_hip.PATH_PER_TOKEN, osm_hip.PATH_GROUPED])
@pytest.mark.parametrize("sublayer", [False, True])
def test_layer_routes_by_rule(ctx, model, router, shared, path, sublayer):
    slab, _, cache, layer = model
    rng = np.random.default_rng(3)
    bias = (0.1 * rng.normal(size=E)).astype(np.float32)
    rule = osm_hip.RouteRule(E, K, **RULE)
    moe = layer(router, shared)
    moe.set_path(path)
    moe.set_routing(rule, bias)
    moe.routing_stats(reset=True)
    for T in (1, 5, 33, 200):
        print(f"[rule layer] T={T}", flush=True)
        x = O.synth_tokens(SEED, 7 * T, T, D)
        xd, yd = ctx.alloc(x.nbytes), ctx.alloc(x.nbytes)
        xd.upload(x)
        moe.decode_device(slab, 0, xd.ptr, yd.ptr, T, sublayer=sublayer)
        y = yd.download(np.float32, T * D).reshape(T, D)
        r = moe.routing(T)
        ids, w, mass = route(r["logits"], rule, bias)
        assert np.array_equal(r["ids"], ids)
        assert np.all(np.abs(r["weights"] - w) <= REL * np.abs(w))
        assert np.all(np.abs(r["mass"] - mass) <= REL * mass)
        # The experts themselves: the same picks given from outside, through the cached path's kernels. Those are the per-token
        # kernels; the grouped path differs by its bf16 terms (16 significant bits of the activations, twice).
        ref = moe.run_cached(cache, 0, x, sublayer=sublayer, picks=(r["ids"], r["weights"]))["out"]
        assert np.array_equal(y, ref) if path == osm_hip.PATH_PER_TOKEN else rel_l2(y, ref) <= 2.0**-15
    assert moe.routing_stats()["selections"] == 1 + 5 + 33 + 200
    # And back: softmax top-k as before the rule.
    x = O.synth_tokens(SEED, 0, 9, D)
    moe.set_routing(None)
    got, ref = moe.run_slab(slab, 0, x, sublayer), layer(router, shared)
    ref.set_path(path)
    ref = ref.run_slab(slab, 0, x, sublayer)
    assert np.array_equal(got["out"], ref["out"]) and np.array_equal(got["ids"], ref["ids"])


def test_rule_on_the_other_paths(ctx, model):
    slab, _, cache, layer = model
    rng = np.random.default_rng(4)
    bias = (0.1 * rng.normal(size=E)).astype(np.float32)
    rule = osm_hip.RouteRule(E, K, **RULE)
    moe = layer()
    moe.set_path(osm_hip.PATH_PER_TOKEN)
    moe.set_routing(rule, bias)
    T = 20
    x = O.synth_tokens(SEED, 1, T, D)
    ref = moe.run_slab(slab, 0, x, sublayer=True)
    assert np.array_equal(ref["ids"], route(ref["logits"], rule, bias)[0])
    # Cached, static and by phases: the same kernels, the same bits.
    got = moe.run_cached(cache, 0, x, sublayer=True)
    assert np.array_equal(got["out"], ref["out"]) and np.array_equal(got["weights"], ref["weights"])
    xd, yd, zd = ctx.alloc(x.nbytes), ctx.alloc(x.nbytes), ctx.alloc(x.nbytes)
    xd.upload(x)
    moe.decode_device_static(slab, 0, xd.ptr, yd.ptr, T, sublayer=True)
    assert np.array_equal(yd.download(np.float32, T * D).reshape(T, D), ref["out"])
    for phase in range(3):
        moe.launch_phase(slab, 0, xd.ptr, zd.ptr, T, True, phase)
    assert np.array_equal(zd.download(np.float32, T * D).reshape(T, D), ref["out"])
    stack = osm_hip.run_cached_layers(ctx, [moe, moe], [0, 0], cache, x)
    two = moe.run_slab(slab, 0, ref["out"], sublayer=True)["out"]
    assert np.array_equal(np.asarray(stack).reshape(T, D), two)
    # A graph, replayed with other inputs and other work between the replays.
    with ctx.capture() as cap:
        moe.decode_device(slab, 0, xd.ptr, yd.ptr, T, sublayer=True)
    for i in range(3):
        xi = O.synth_tokens(SEED, 100 * i, T, D)
        xd.upload(xi)
        cap.graph.launch()
        y = yd.download(np.float32, T * D).reshape(T, D)
        assert np.array_equal(y, moe.run_slab(slab, 0, xi, sublayer=True)["out"])
    # A bf16 prompt chunk.
    moe.set_path(osm_hip.PATH_AUTO)
    T = 100
    xb = bf16_bits(O.synth_tokens(SEED, 3, T, D))
    xd2, yd2 = ctx.alloc(xb.nbytes), ctx.alloc(T * D * 4)
    xd2.upload(xb)
    moe.prefill_device(slab, 0, xd2.ptr, yd2.ptr, T)
    r = moe.routing(T)
    assert np.array_equal(r["ids"], route(r["logits"], rule, bias)[0])
    ref = moe.run_cached(cache, 0, bf16_to_f32(xb), picks=(r["ids"], r["weights"]))["out"]
    assert rel_l2(yd2.download(np.float32, T * D).reshape(T, D), ref) <= 2.0**-15


def test_refused_layer_rules(ctx, model):
    moe = model[3]()
    for rule, bias in ((osm_hip.RouteRule(32, K), None), (osm_hip.RouteRule(E, K + 1), None),
                       (osm_hip.RouteRule(E, K, groups=7), None), (osm_hip.RouteRule(E, K), np.full(E, np.nan))):
        with pytest.raises(osm_hip.OsmError) as e:
            moe.set_routing(rule, bias)
        assert e.value.status == osm_hip.OSM_E_INVALID
    with pytest.raises(ValueError):
        moe.set_routing(osm_hip.RouteRule(E, K), np.zeros(E - 1))
    a = ctx.alloc(256)
    a.upload(np.zeros(64, np.int32))
    with ctx.capture():
        with pytest.raises(osm_hip.OsmError) as e:
            moe.set_routing(osm_hip.RouteRule(E, K), np.zeros(E))
        osm_hip.group_rows(ctx, a.ptr, 8, 2, a.ptr.value + 64, a.ptr.value + 128)  # the capture goes on
    assert "capture" in e.value.diagnostic
