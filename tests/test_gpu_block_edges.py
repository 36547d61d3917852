"""Calls of the operators around an expert layer that the first tests of them
did not make: rows of nothing but NaN, empty pairs with weights that are no
numbers, biases with strides, scratch between captured calls, outputs that lie
beside their inputs, and a routing rule under the streaming lookahead.

Tolerances.  u = 2^-24.  Routing weights: expf of 2 ulp (4 u) on an argument
whose rounding is taken back, a sum of at most 32 of them in five levels (5 u
relative, all terms positive) with 4 u of its own terms, one division (correctly
rounded, u), the scale (u): below 20 u, and 32 u is taken, as for every routing
test.  Everything else is compared bit for bit."""
import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from test_gpu_block import (BF16, F16, F32, H, U, check_route, close, d64, randn, route_ref,  # noqa: E402
                            router_logits)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


# ---- routing -------------------------------------------------------------------

@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups", [(1, 1, 1), (4, 2, 1), (4, 2, 2)])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_rows_without_a_number(score, bias, groups, renorm):
    """Rows of NaN, of NaN and -inf, of NaN and +inf: the weights are NaN where
    the formula's are, renormalised or not."""
    E, inf = 48, math.inf
    x = 2 * randn(6, E, seed=3)
    x[0] = math.nan
    x[1] = math.nan
    x[1, ::2] = -inf
    x[2] = -inf
    x[2, E - 1] = math.nan
    x[3] = math.nan
    x[3, 5] = inf
    x[4] = -inf
    b = 0.1 * randn(E, seed=4) if bias else None
    check_route(x, 6, score=score, bias=b, n_group=groups[0], topk_group=groups[1], group_top=groups[2], renorm=renorm)


def masked_ref(logits, k, score="softmax", bias=None, n_group=1, topk_group=1, group_top=1, renorm=True, scale=1.0):
    """A masked rule token by token in 64 bits: an expert whose logit is -inf
    (or NaN) compares as -inf, a group's sum has only what is left of it."""
    L = logits.double().cpu().numpy()
    b = np.zeros(L.shape[1]) if bias is None else bias.double().cpu().numpy()
    ids, ws = [], []
    with np.errstate(all="ignore"):
        for l in L:
            off = np.isneginf(l) | np.isnan(l)
            e = np.exp(l - l.max()) if np.isfinite(l.max()) else np.zeros_like(l)
            s = 1 / (1 + np.exp(-l)) if score == "sigmoid" else e / e.sum() if e.sum() else e
            by_logit = bias is None and (n_group == 1 or group_top == 1)
            c = np.where(off, -np.inf, l if by_logit else s + b)
            per = len(l) // n_group
            strength = []
            for g in range(n_group):
                best = sorted(c[g * per:(g + 1) * per], reverse=True)[:group_top]
                strength.append(sum(v for v in best if v > -np.inf) if best[0] > -np.inf else -np.inf)
            keep = sorted(range(n_group), key=lambda g: (-strength[g], g))[:topk_group]
            pick = sorted((i for i in range(len(l)) if i // per in keep), key=lambda i: (-c[i], i))[:k]
            w = s[pick]
            if renorm:
                w = w / w.sum() if w.sum() else 0 * w
            ids.append(pick)
            ws.append(w * np.float64(np.float32(scale)))
    return torch.tensor(np.array(ids)), torch.tensor(np.array(ws))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [None, 0.5, -5.0])
@pytest.mark.parametrize("E,k,groups", [(48, 6, (1, 1, 1)), (48, 6, (4, 2, 1)), (48, 6, (4, 2, 2)), (157, 6, (1, 1, 1)),
                                        (256, 8, (4, 2, 2)), (512, 16, (1, 1, 1)), (493, 5, (17, 3, 2)), (32, 4, (32, 8, 2))])
def test_masked_experts_are_chosen_last(score, bias, E, k, groups):
    """Under a positive bias no expert that a token may not use is chosen while
    others are left, in every layout of the lanes; rows with one, with none and
    with all experts left."""
    from moe_prefetch_b200 import Routing
    n = 65
    x = 2 * randn(n, E, seed=E)
    g = torch.Generator().manual_seed(E)
    x.scatter_(1, torch.randint(0, E, (n, max(1, E // 3)), generator=g).cuda(), -math.inf)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, E // 2] = 1.0
    x[2] = 2 * randn(E, seed=1)
    x[3, E // 2:] = -math.inf
    b = None if bias is None else bias + 0.2 * randn(E, seed=2)
    kw = dict(score=score, bias=b, n_group=groups[0], topk_group=groups[1], group_top=groups[2], scale=1.5)
    for renorm in (True, False):
        ids, w = Routing(E, k, masked=True, renorm=renorm, **kw)(x)
        rid, rw = masked_ref(x, k, renorm=renorm, **kw)
        assert torch.equal(ids.long().cpu(), rid)
        close(w, rw, 32 * U * rw.abs(), "w")
    if groups[0] == 1:
        left = torch.isfinite(x).sum(1, keepdim=True).clamp(max=k).cpu()
        off = torch.isneginf(x).gather(1, ids.long()).cpu()
        assert torch.equal(off, torch.arange(k)[None] >= left)


def test_a_layer_takes_a_masked_rule():
    """A rule with masks on a layer whose logits have none: the plain rule."""
    from moe_prefetch_b200 import MoeStack, Routing
    st = MoeStack(n_layers=1, n_expert=64, n_ff=256)
    try:
        st.synth_resident(seed=2)
        x, b = randn(5, H, seed=1), 0.2 * randn(64, seed=2)
        got = []
        for masked in (False, True):
            st.set_routing(0, Routing(64, 8, score="sigmoid", bias=b, n_group=4, topk_group=2, group_top=2, masked=masked))
            got.append(st.layer_forward(0, x))
        assert all(torch.equal(p, q) for p, q in zip(*got))
    finally:
        st.close()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("scale", [1.0, 1.5])
def test_weights_of_far_logits(score, renorm, scale):
    """Scores that underflow in 32 bits beside a small sum: every weight is
    within 32 u of its value, or two steps of the smallest fp32 (one rounding
    there, and one of its product with the scale)."""
    from moe_prefetch_b200 import Routing
    E, k = 64, 8
    x = torch.full((40, E), -300.0)
    for t in range(40):        # the bias decides: the chosen are 40 to 103 below the largest, or below 0
        x[t, :k] = -40.0 - 1.6 * t - 6.0 * torch.arange(k)
        x[t, k - 1] = -103.0
    x[:, E - 1] = 0.0
    x[5, :k] = -20.0 * torch.arange(k) - 10.0
    x[6, :k] = torch.tensor([-87.0, -88.5, -88.9, -90.0, -95.0, -100.0, -103.0, -110.0])
    b = torch.zeros(E)
    b[:k] = 4.0 + torch.arange(k) / 16
    x, b = x.cuda(), b.cuda()
    ids, w = Routing(E, k, score=score, bias=b, renorm=renorm, scale=scale)(x)
    rid, rw = route_ref(x, k, score=score, bias=b, renorm=renorm, scale=scale)
    assert torch.equal(ids.long().cpu(), rid)
    err = (d64(w) - rw).abs()
    assert (err <= 32 * U * rw + 2 * 2.0 ** -149).all(), (err / rw.clamp(min=1e-300)).max()


# ---- outputs beside and over inputs ---------------------------------------------------

def test_outputs_between_the_rows_of_inputs():
    """r, y, r' and x as columns of one buffer: the bits of separate tensors."""
    from moe_prefetch_b200 import BlockNorm
    n, h = 400, 256
    buf = randn(n, 4 * h, seed=1)
    r, y, ro, x = (buf[:, i * h:(i + 1) * h] for i in range(4))
    nm = BlockNorm(h, post=1 + 0.2 * randn(h, seed=2), pre=True, scale=0.5)
    want = nm(r.contiguous(), y.contiguous())
    got = nm(r, y, out=(ro, x))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("h", [64, 2048, 1537, 8200])
def test_outputs_over_every_input_of_a_row(h):
    """r' over y and x over r, x over a full gate, r' over add: the bits of
    separate tensors."""
    from moe_prefetch_b200 import BlockNorm
    n, k = 300, 2
    r, y, gate = (randn(n, h, seed=s) for s in (1, 2, 3))
    nm = BlockNorm(h, post=1 + 0.2 * randn(h, seed=4), pre=True, gate_act="sigmoid", scale=0.5)
    want = nm(r, y, gate=gate)
    for pick in (lambda r, y, g: (y, r), lambda r, y, g: (r, g), lambda r, y, g: (g, y)):
        t = [v.clone() for v in (r, y, gate)]
        got = nm(t[0], t[1], gate=t[2], out=pick(*t))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    pos = torch.randperm(n * k, generator=torch.Generator().manual_seed(5)).int().view(n, k).cuda()
    rows, w, add = randn(n * k, h, seed=6), randn(n, k, seed=7), randn(n, h, seed=8)
    want = nm.combine(r, rows, pos, w, add=add, gate=gate)
    t = [v.clone() for v in (r, add, gate)]
    got = nm.combine(t[0], rows, pos, w, add=t[1], gate=t[2], out=(t[1], t[2]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_block_refuses_overlaps():
    """Through a context: y on x, r' or x' shifted against x or r, ids on w."""
    from moe_prefetch_b200 import BlockNorm, MoeStack, _lib
    st = MoeStack(n_layers=1, n_expert=64, n_ff=256)
    try:
        st.synth_resident(seed=1)
        n = 3
        buf = torch.zeros(8 * n * H, device="cuda")
        part = lambda i, shift=0: C.c_void_p(buf.data_ptr() + 4 * (i * n * H + shift))
        ids, w = torch.zeros(n, 8, dtype=torch.int32, device="cuda"), torch.zeros(n, 8, device="cuda")
        nm = BlockNorm(H, pre=True)

        def rc(x, y=None, r=None, ro=None, xo=None, i=ids.data_ptr(), ww=w.data_ptr(), gate=None):
            b = _lib.MoeBlock()
            if y is None:
                b.norm, b.r, b.r_out, b.x_out = C.pointer(nm.with_gate(gate, n, F32, ids.device)), r, ro, xo
            return st.lib.moe_block_forward(st.ctx, 0, x, n, C.byref(b), y, C.c_void_p(i), C.c_void_p(ww), 0, None)

        assert rc(part(0), y=part(1)) == 0
        assert rc(part(0), r=part(1), ro=part(1), xo=part(0)) == 0
        assert rc(part(0), r=part(1), ro=part(2), xo=part(3)) == 0
        for bad in (dict(y=part(0)), dict(y=part(0, 64)), dict(y=part(1), i=w.data_ptr()), dict(y=part(1), i=buf.data_ptr()),
                    dict(y=part(1), ww=buf.data_ptr() + 4 * n * H), dict(r=part(1), ro=part(1, 8), xo=part(3)),
                    dict(r=part(1), ro=part(2), xo=part(2, 8)), dict(r=part(1), ro=part(2), xo=part(0, 4)),
                    dict(r=part(1), ro=part(2), xo=C.c_void_p(ids.data_ptr())),
                    dict(r=part(1), ro=part(2), xo=part(3), i=buf.data_ptr() + 4 * n * H),
                    dict(r=part(1), ro=part(2), xo=part(3), gate=w[:, :1])):
            assert rc(part(0), **bad) == -1, bad
        torch.cuda.synchronize()
    finally:
        st.close()


# ---- norms -----------------------------------------------------------------------

@pytest.mark.parametrize("h", [64, 2048, 1537, 1026, 8200, 16384])   # registers, odd, pairs, shared memory
@pytest.mark.parametrize("weight", [math.nan, math.inf, -math.inf])
def test_combine_empty_pairs_add_nothing(h, weight):
    """A pos outside y_rows adds nothing, whatever its weight: the bits of the
    same call with weight 0 there."""
    from moe_prefetch_b200 import BlockNorm
    n, k = 5, 3
    rows, r = randn(n * k, h, seed=1), randn(n, h, seed=2)
    pos = torch.arange(n * k, dtype=torch.int32).view(n, k)
    pos[0, 0], pos[1, 2], pos[2, 1] = -1, n * k, -7
    pos[3] = -1
    empty = ((pos < 0) | (pos >= n * k)).cuda()
    w = torch.rand(n, k, generator=torch.Generator().manual_seed(3)).cuda()
    nm = BlockNorm(h, post=1 + 0.2 * randn(h, seed=4), pre=True)
    want = nm.combine(r, rows, pos.cuda(), w.masked_fill(empty, 0.0))
    got = nm.combine(r, rows, pos.cuda(), w.masked_fill(empty, weight))
    assert torch.isfinite(want[0]).all() and torch.isfinite(want[1]).all()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- adapters ----------------------------------------------------------------------

@pytest.mark.parametrize("wt,parts", [(BF16, 2.0 ** -26), (F16, 2.0 ** -23)])
@pytest.mark.parametrize("n", [40, 3000])     # both tile sizes
def test_fp32_rows_keep_their_bits(n, wt, parts):
    """One weight of 1 in A and in B: out is x as the two products see it.  hi is
    off by half a step of 11 bits and lo is cut off at 11 bits below: 2^-22 of x;
    A x = hi + lo has 23 bits, exact in fp32, and is split into parts that leave
    out 2^-26 (three of bf16) or 2^-23 (two of fp16); their sum is exact."""
    from moe_prefetch_b200 import AdapterSet
    a, b = torch.zeros(1, 8, 64, dtype=wt).cuda(), torch.zeros(1, 16, 8, dtype=wt).cuda()
    a[0, 3, 17], b[0, 5, 3] = 1.0, 1.0
    x = torch.zeros(n, 64).cuda()
    x[:, 17] = randn(n, seed=n)
    out = AdapterSet(a, b)(x, torch.zeros(n, dtype=torch.int32, device="cuda"))
    got, want = d64(out[:, 5]), d64(x[:, 17])
    assert ((got - want).abs() <= (2.0 ** -22 + parts) * want.abs()).all(), ((got - want) / want).abs().max()


@pytest.mark.parametrize("wt", [BF16, F16])
@pytest.mark.parametrize("at", ["a", "b"])
def test_fp32_rows_of_the_largest_values(wt, at):
    """Finite values up to the largest stay finite (2^-21 there), in x and in A x."""
    from moe_prefetch_b200 import AdapterSet
    a, b = torch.zeros(1, 1, 64, dtype=wt).cuda(), torch.zeros(1, 16, 1, dtype=wt).cuda()   # (rank 1: no 0 * inf)
    a[0, 0, 1], b[0, 0, 0] = (2.0 ** -14, 1.0) if at == "a" else (1.0, 2.0 ** -14)
    v = torch.tensor([torch.finfo(F32).max, -torch.finfo(F32).max, 2.0 ** 127, 2.0 ** 127 - 2.0 ** 103, 3.4e38, math.inf, math.nan])
    x = torch.zeros(7, 64)
    x[:, 1] = v
    out = d64(AdapterSet(a, b)(x.cuda(), torch.zeros(7, dtype=torch.int32, device="cuda"))[:, 0])
    want = d64(v) * 2.0 ** -14
    assert ((out - want).abs()[:5] <= (2.0 ** -21 + 2.0 ** -23) * want.abs()[:5]).all()
    assert out[5] == math.inf and torch.isnan(out[6])


# ---- a rule under the streaming lookahead ---------------------------------------------

def test_stream_lookahead_goes_by_the_rule():
    """Layer 1 routes by bias and groups.  What the lookahead of layer 0
    streams into layer 1, and what layer 1 then routes to, are experts of its
    rule: with the same input on both layers nothing else ever becomes
    resident there, and streamed experts are found in time."""
    import time
    from moe_prefetch_b200 import MoeCacheConfig, MoeStack, Routing
    E, K, L = 128, 8, 2
    src = MoeStack(n_layers=L, n_expert=E, n_ff=256)
    src.synth_resident(seed=71, keep_router=True)
    host = [tuple(v[:E].contiguous().cpu().pin_memory() for v in src.slot_views(il)) for il in range(L)]
    routers = [r.clone() for r in src.routers]
    st = MoeStack(n_layers=L, n_expert=E, n_ff=256, cache=MoeCacheConfig(
        n_slots=64, max_inserts=8, admit="off", batch_tables=True, early_issue=True, stream=True, stream_per_layer=8,
        stream_reserve=4))
    # the bias turns the order of the logits around: the experts with the largest ones are never chosen
    bias = 0.3 * randn(E, seed=9)
    kw = dict(score="sigmoid", bias=bias, n_group=8, topk_group=3, group_top=2)
    try:
        for il in range(L):
            st.set_router(il, routers[il])
            st.set_expert_weights(il, *host[il])
        src.routers = routers
        st.set_routing(1, Routing(E, K, **kw))
        allowed, raw = set(), set()
        for t in range(12):
            x = randn(1, H, seed=200 + t)
            lg = router_logits(src, 1, x)
            rid, _ = route_ref(lg, K, **kw)
            allowed |= set(rid[0].tolist())
            raw |= set(lg[0].topk(K)[1].tolist())
            for il in range(L):
                _, ids, _ = st.layer_forward(il, x)
                torch.cuda.synchronize()
                time.sleep(0.001)
            assert torch.equal(ids.long().cpu(), rid)
            st.step()
        torch.cuda.synchronize()
        st.step()
        resident = st.tables(1)["slot_expert"]
        resident = set(int(e) for e in resident[resident >= 0])
        ss = st.stream_stats()
        assert raw - allowed                       # (the two rules differ on these inputs)
        assert ss["words"] > 0 and resident
        assert resident <= allowed, sorted(resident - allowed)
        assert ss["in_time"] > 0, ss
    finally:
        st.close()
        src.close()


# ---- scratch between captured calls ------------------------------------------------------

def test_one_plain_call_makes_room_for_every_captured_one():
    """The largest n_tok once, without adapters.  Then calls with router
    adapters, with layer adapters and with both are captured and replayed
    between eager calls of the other kinds: none allocates, and every replay has
    the eager call's bits."""
    from moe_prefetch_b200 import AdapterSet, BlockNorm, MoeStack
    st = MoeStack(n_layers=1, n_expert=64, n_ff=256)
    try:
        st.synth_resident(seed=3)
        n = 24
        x, r = randn(n, H, seed=1), randn(n, H, seed=2)
        ids = torch.randint(-1, 3, (n,), generator=torch.Generator().manual_seed(4)).int().cuda()
        ra = AdapterSet((randn(3, 8, H, seed=5) / 45).to(BF16), randn(3, 64, 8, seed=6).to(BF16))
        la = AdapterSet((randn(3, 8, H, seed=7) / 45).to(BF16), randn(3, H, 8, seed=8).to(BF16))
        nm = BlockNorm(H, post=1 + 0.2 * randn(H, seed=9), pre=True)
        st.block_forward(0, x)
        torch.cuda.synchronize()
        calls = [lambda kw=kw, m=m: st.block_forward(0, x[:m], r=r[:m], norm=nm, adapter_ids=ids[:m], **kw)
                 for kw, m in ((dict(router_adapters=ra), n), (dict(adapters=la), n - 1),
                               (dict(router_adapters=ra, adapters=la), n))]
        graphs = []
        for call in calls:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = call()
            graphs.append((g, out))
        for turn in range(2):
            x.copy_(randn(n, H, seed=20 + turn))
            want = [call() for call in calls]
            for (g, out), w in zip(graphs, want):
                g.replay()
                assert all(torch.equal(a, b) for a, b in zip(out, w))
        torch.cuda.synchronize()
    finally:
        st.close()


# ---- arguments -------------------------------------------------------------------------

@pytest.fixture(scope="module")
def one_layer():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from moe_prefetch_b200 import MoeStack
    st = MoeStack(n_layers=1, n_expert=64, n_ff=256)
    st.synth_resident(seed=6, keep_router=True)
    yield st
    st.close()


def test_route_bias_with_a_stride_is_read_at_every_call():
    from moe_prefetch_b200 import Routing
    E = 64
    table = 0.3 * randn(E, 3, seed=1)
    x = randn(9, E, seed=2)
    rt = Routing(E, 4, score="sigmoid", bias=table[:, 1])
    for turn in range(2):
        ids, w = rt(x)
        rid, rw = route_ref(x, 4, score="sigmoid", bias=table[:, 1])
        assert torch.equal(ids.long().cpu(), rid)
        table.copy_(0.3 * randn(E, 3, seed=7))


def test_layer_rule_takes_a_bias_with_a_stride(one_layer):
    from moe_prefetch_b200 import Routing
    bias = 0.3 * randn(64, 2, seed=3)[:, 1]
    x = randn(4, H, seed=4)
    rid, _ = route_ref(router_logits(one_layer, 0, x), 8, score="sigmoid", bias=bias)
    one_layer.set_routing(0, Routing(64, 8, score="sigmoid", bias=bias))
    try:
        assert torch.equal(one_layer.layer_forward(0, x)[1].long().cpu(), rid)
    finally:
        one_layer.set_routing(0, None)


def test_outputs_in_a_list_on_a_stream():
    """out as a list, with a stream of the call's own."""
    from moe_prefetch_b200 import BlockNorm, Routing
    x, r = randn(7, 64, seed=1), randn(7, 64, seed=2)
    rt, nm = Routing(64, 4), BlockNorm(64, pre=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = [torch.empty(7, 4, dtype=torch.int32, device="cuda"), torch.empty(7, 4, device="cuda")]
    ro = [torch.empty_like(r), torch.empty_like(r)]
    co = [torch.empty_like(r), torch.empty_like(r)]
    pos, w = torch.arange(7, dtype=torch.int32, device="cuda").view(7, 1), torch.ones(7, 1, device="cuda")
    torch.cuda.synchronize()
    rt(x, out=out, stream=s)
    nm(r, x, out=ro, stream=s)
    nm.combine(r, x, pos, w, out=co, stream=s)
    s.synchronize()
    for got, want in ((out, rt(x)), (ro, nm(r, x)), (co, nm.combine(r, x, pos, w))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- long strides, first calls, captured rules ------------------------------------------

def test_rows_past_32_bits():
    """Rows so far apart that their offsets pass 2^32 elements and bytes."""
    from moe_prefetch_b200 import AdapterSet, BlockNorm, Routing
    n, ld = 36, (1 << 27) + 64             # 36 * 2^27 elements of 16 bits: 9.7 GB, of which little is touched
    big = torch.empty(n * ld, dtype=BF16, device="cuda").view(n, ld)
    cols = [big[:, 64 * i:64 * (i + 1)] for i in range(5)]
    r, y, x = (randn(n, 64, seed=s).to(BF16) for s in (1, 2, 3))
    for c, v in zip(cols, (r, y, x)):
        c.copy_(v)
    rt = Routing(64, 4, score="sigmoid", bias=0.1 * randn(64, seed=4))
    assert all(torch.equal(a, b) for a, b in zip(rt(cols[0]), rt(r)))
    nm = BlockNorm(64, post=1 + 0.2 * randn(64, seed=5), pre=True)
    want = nm(r, y)
    nm(cols[0], cols[1], out=(cols[3], cols[4]))
    assert torch.equal(cols[3], want[0]) and torch.equal(cols[4], want[1])
    st = AdapterSet((randn(3, 8, 64, seed=6) / 8).to(BF16), randn(3, 64, 8, seed=7).to(BF16))
    ids = (torch.arange(n, device="cuda") % 4 - 1).int()
    want = st(x, ids, y)
    assert torch.equal(st(cols[2], ids, cols[1], out=cols[3]), want)
    assert torch.equal(st(cols[2], ids, cols[1], out=cols[1]), want)
    f32 = big.view(F32)                    # combine: expert rows past 2^31 elements
    rows = f32[:, 1024:1088]
    rows.copy_(randn(n, 64, seed=8))
    pos, w = torch.randperm(n, generator=torch.Generator().manual_seed(9)).int().view(n // 2, 2).cuda(), randn(n // 2, 2, seed=10)
    got = nm.combine(r[:n // 2].float(), rows, pos, w)
    want = nm.combine(r[:n // 2].float(), rows.contiguous(), pos, w)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


FIRST = """
import torch
from moe_prefetch_b200 import AdapterSet, BlockNorm, Routing
torch.manual_seed(1)
randn = lambda *s: torch.randn(*s, device="cuda")
rt = Routing(128, 8, score="sigmoid", bias=randn(128), n_group=4, topk_group=2, group_top=2)
nm, wide = BlockNorm(2048, post=randn(2048), pre=True), BlockNorm(16384, post=randn(16384), pre=True)
st = AdapterSet(randn(4, 64, 2048).bfloat16() / 45, randn(4, 256, 64).bfloat16())
lg, r, y, rw, yw, out = randn(300, 128), randn(300, 2048), randn(300, 2048), randn(3, 16384), randn(3, 16384), randn(300, 256)
gate = randn(1, 1).expand(300, 1)
ids = (torch.arange(300, device="cuda") % 5 - 1).int()
pos, w = torch.randint(-1, 300, (300, 4), device="cuda").int(), randn(300, 4)
call = lambda: [*rt(lg), *nm(r, y, gate=gate), *wide(rw, yw), *nm.combine(r, y, pos, w), st(y, ids, out)]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = call()
g.replay()
want = call()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("captured")
"""


def test_first_calls_of_a_process_can_be_captured():
    """Nothing has to run before a capture: neither a kernel's first launch nor
    its shared memory limit."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("n", [1, 6])
def test_captured_layers_keep_their_rule(one_layer, n):
    """A captured call of a layer with a rule gives the rule's results after
    the layer has another."""
    from moe_prefetch_b200 import Routing
    x = randn(n, H, seed=1)
    one_layer.set_routing(0, Routing(64, 8, score="sigmoid", n_group=8, topk_group=3, group_top=2, renorm=False))
    try:
        one_layer.block_forward(0, x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = one_layer.block_forward(0, x)
        x.copy_(randn(n, H, seed=2))
        want = one_layer.block_forward(0, x)
    finally:
        one_layer.set_routing(0, None)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not torch.equal(one_layer.block_forward(0, x)[2], want[2])
