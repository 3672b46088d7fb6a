"""The operators of batches together, as a server of many requests runs them:
each token's hidden row through a projection with its request's adapter, the
result through a layer that routes by a rule, and the picks grouped by expert
and by request."""

import numpy as np
import pytest

import oracle as O
import osm_hip
from rule_reference import route
from test_gpu_q4_project import BF16, F32, Problem

pytestmark = pytest.mark.gpu

SEED, D, I, G, E, K = 29, 512, 128, 64, 64, 6


@pytest.mark.parametrize("T", [1, 23, 160])
def test_projection_routing_grouping(ctx, T):
    g = osm_hip.geometry(D, I, G, osm_hip.BF16)
    slab = osm_hip.ExpertSlab(ctx, g, 1, E)
    slab.synthesize(SEED)
    moe = osm_hip.MoeLayer(ctx, g, E, K, O.synth_router_bf16(SEED, 0, E, D), osm_hip.BF16, O.synth_shared_gate_bf16(SEED, 0, D),
                           O.synth_norm_weight(SEED, 0, D), O.synth_expert_blob(SEED, 0, O.SHARED_EXPERT_ID, D, I, G), max_tokens=T)
    rule = osm_hip.RouteRule(E, K, osm_hip.SCORE_SIGMOID, groups=8, top_groups=4, group_score=2, scale=2.5)
    bias = (0.1 * np.random.default_rng(1).normal(size=E)).astype(np.float32)
    moe.set_routing(rule, bias)
    p = Problem(ctx, T, D, 256, 64, BF16, F32, count=5, rank=8)
    y, lg, ids, w = (ctx.alloc(4 * T * n) for n in (D, E, K, K))
    b, off, order = ctx.alloc(4 * E), ctx.alloc(4 * (E + 1)), ctx.alloc(4 * T * K)
    req_off, req_order = ctx.alloc(4 * 6), ctx.alloc(4 * T)
    b.upload(bias)

    def step():
        p.call()
        moe.decode_device(slab, 0, p.yd.ptr, y.ptr, T, sublayer=True)
        osm_hip.route_experts(ctx, rule, lg.ptr, F32, T, ids.ptr, w.ptr, bias_ptr=b.ptr)
        osm_hip.group_rows(ctx, ids.ptr, T * K, E, off.ptr, order.ptr)
        osm_hip.group_rows(ctx, p.dev[4].ptr, T, 5, req_off.ptr, req_order.ptr)

    step()  # grows the workspaces; the logits that route_experts takes are filled next
    h = p.yd.download(np.float32, T * D).reshape(T, D)
    assert np.all(np.abs(h - p.y64) <= p.tol)
    r = moe.routing(T)
    lg.upload(r["logits"])
    with ctx.capture() as cap:
        step()
    eager = None
    for _ in range(3):
        for a in (y, ids, w, off, order, req_off, req_order):
            a.upload(np.zeros(a.nbytes, np.uint8))
        cap.graph.launch()
        got = [a.download(np.uint32, a.nbytes // 4) for a in (y, ids, w, off, order, req_off, req_order)]
        if eager is None:
            step()
            eager = [a.download(np.uint32, a.nbytes // 4) for a in (y, ids, w, off, order, req_off, req_order)]
        assert all(np.array_equal(x, z) for x, z in zip(got, eager))
    rid, _, _ = route(r["logits"], rule, bias)
    assert np.array_equal(eager[1].reshape(T, K), rid) and np.array_equal(r["ids"], rid)
    assert np.array_equal(eager[2].view(np.float32).reshape(T, K), r["weights"])
    assert np.array_equal(eager[4], np.argsort(rid.reshape(-1), kind="stable"))
    assert np.array_equal(eager[3], np.searchsorted(np.sort(rid.reshape(-1)), np.arange(E + 1)))
    key = np.where(p.ids < 0, 5, p.ids)
    assert np.array_equal(eager[6], np.argsort(key, kind="stable"))
