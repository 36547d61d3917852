"""The operators around an expert layer against their formulas in 64 bits, at
the sizes, types, strides and masks where they can go wrong, and the whole
block through MoeStack.

Tolerances.  u = 2^-24 is fp32's rounding; an output of another type adds its
own half step, finfo.eps / 2.  Routing: ids equal; weights are formed in 64
bits and rounded once, except that a softmax without renormalisation divides
by a sum in fp32 (per term: 2 ulp of expf and one rounding of l - max, at most
e^-d * d <= 0.37 ulp of the largest term; then at most 16 + 5 additions): 32 u.
Norms: a mean of squares of up to 16 * 32 * 32 values in chains of 16, 5 and 5
additions, half of which enters the root, then five roundings: 32 u of each
term.  Adapters: chains of at most n / 8 additions, each of one rounding or, on
the tensor cores, one truncation of the partial sum (2 u): (n / 8 + 32) * 2 u
of the sum of absolute terms, for each of the two products.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}


@pytest.fixture(autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def close(got, want, bound, what):
    """|got - want| <= bound + the output type's half step, everywhere."""
    got64 = got.double().cpu()
    lim = bound + HALF[got.dtype] * (want.abs() + bound) + TINY[got.dtype]
    bad = ~((got64 - want).abs() <= lim)
    bad &= ~(torch.isnan(got64) & torch.isnan(want)) & ~(got64 == want)
    assert not bad.any(), (what, int(bad.sum()), (got64 - want).abs()[bad].max().item(), lim[bad].min().item())


# ---- routing -------------------------------------------------------------------

def route_ref(logits, k, score="softmax", bias=None, n_group=1, topk_group=1, group_top=1, renorm=True, scale=1.0,
              prior=None):
    """The rule token by token in 64 bits (numpy): ids, w."""
    L = logits.double().cpu().numpy()
    n, E = L.shape
    b = None if bias is None else bias.double().cpu().numpy()
    ids, ws = np.zeros((n, k), np.int64), np.zeros((n, k))
    with np.errstate(all="ignore"):
        for t in range(n):
            l = L[t]
            if score == "sigmoid":
                s = 1.0 / (1.0 + np.exp(-l))
            else:
                m = l.max() if not np.isnan(l).any() else np.nan
                e = np.zeros(E) if m == -np.inf else np.exp(l - m)
                tot = e.sum()
                s = np.zeros(E) if tot == 0 else e / tot
            by_logit = b is None and prior is None and (n_group == 1 or group_top == 1)
            c = l.copy() if by_logit else s if b is None else s + b
            c = np.where(np.isnan(c), -np.inf, c)
            alive = np.ones(E, bool)
            per = E // n_group
            if n_group > 1:
                gs = []
                for g in range(n_group):
                    top = sorted(c[g * per:(g + 1) * per], reverse=True)[:min(group_top, per)]
                    v = top[0] + top[1] if len(top) == 2 else top[0]
                    gs.append(-np.inf if np.isnan(v) else v)
                for g in sorted(range(n_group), key=lambda g: (-gs[g], g))[topk_group:]:
                    alive[g * per:(g + 1) * per] = False
            if prior is not None:
                c = c + prior
            pick = sorted((e for e in range(E) if alive[e]), key=lambda e: (-c[e], e))[:k]
            w = s[pick]
            if renorm:
                tot = w.sum()
                w = np.zeros(k) if tot == 0 else w / tot
            ids[t], ws[t] = pick, w * np.float64(np.float32(scale))
    return torch.from_numpy(ids), torch.from_numpy(ws)


def check_route(logits, k, **kw):
    from moe_prefetch_b200 import Routing
    ids, w = Routing(logits.shape[1], k, **kw)(logits)
    rid, rw = route_ref(logits, k, **kw)
    assert torch.equal(ids.long().cpu(), rid)
    close(w, rw, 32 * U * rw.abs(), "w")


def randn(*shape, seed=0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("E,k,n_group,topk_group", [
    (1, 1, 1, 1), (5, 5, 1, 1), (32, 8, 1, 1), (128, 8, 1, 1), (157, 6, 1, 1), (256, 8, 4, 2), (256, 8, 8, 3),
    (512, 32, 1, 1), (512, 16, 3, 2), (510, 7, 3, 1), (480, 9, 5, 2), (504, 4, 9, 4), (493, 5, 17, 3), (64, 8, 32, 4),
    (96, 3, 32, 32), (24, 24, 6, 6)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("rule", ["plain", "bias", "norenorm"])
def test_route(E, k, n_group, topk_group, score, rule):
    if E % n_group:
        pytest.skip("groups do not divide")
    bias = 0.1 * randn(E, seed=1) if rule == "bias" else None
    for n, dtype, top in ((1, F32, 2), (37, BF16, 1), (130, F16, 2)):
        x = (2.0 * randn(n, E, seed=E + n)).to(dtype)
        check_route(x, k, score=score, bias=bias, n_group=n_group, topk_group=topk_group, group_top=top,
                    renorm=rule != "norenorm", scale=1.5)


def nextafter(x, steps):
    return (x.view(torch.int32) + steps).view(F32)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_close_and_equal_scores(score, bias):
    """Logits one fp32 step apart, equal ones, and -0 beside +0: the order is
    the exact one, ties to the lower index."""
    E = 64
    x = torch.full((3, E), 3.0).cuda()
    x[0] = nextafter(torch.full((E,), 3.0), torch.randperm(E, generator=torch.Generator().manual_seed(2)).int()).cuda()
    x[1, ::2] = -0.0
    x[1, 1::2] = 0.0
    b = torch.full((E,), 0.25).cuda() if bias else None
    check_route(x, 9, score=score, bias=b)
    check_route(x, 9, score=score, bias=b, n_group=4, topk_group=2, group_top=2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups", [(1, 1, 1), (4, 2, 1), (4, 2, 2)])
def test_route_masks(score, bias, groups):
    """-inf, +inf, NaN, the lowest value and rows with nothing left."""
    E, inf, low = 48, math.inf, torch.finfo(F32).min
    x = 2 * randn(9, E, seed=3)
    x[0] = -inf
    x[1, 1:] = -inf
    x[2, ::3] = low
    x[3] = low
    x[4, 7] = inf
    x[5, 5] = math.nan
    x[6, 20:24] = math.nan
    x[7, :40] = -inf
    x[8] = 1000 * x[8]
    b = 0.1 * randn(E, seed=4) if bias else None
    for renorm in (True, False):
        check_route(x, 6, score=score, bias=b, n_group=groups[0], topk_group=groups[1], group_top=groups[2],
                    renorm=renorm)
    if bias:
        b2 = b.clone()
        b2[3], b2[9], b2[11] = -inf, inf, math.nan
        check_route(x, 6, score=score, bias=b2, n_group=groups[0], topk_group=groups[1], group_top=groups[2])


def test_route_strides_out_stream_graph():
    from moe_prefetch_b200 import Routing
    big = randn(33, 200, seed=5)
    view = big[:, 8:136]
    rt = Routing(128, 8, score="sigmoid", bias=0.1 * randn(128, seed=6), n_group=4, topk_group=2, group_top=2)
    ids, w = rt(view)
    rid, rw = rt(view.contiguous())
    assert torch.equal(ids, rid) and torch.equal(w, rw)
    out = (torch.full((40, 8), -5, dtype=torch.int32, device="cuda"), torch.full((40, 8), -5.0, device="cuda"))
    got = rt(view, out=(out[0][:33], out[1][:33]))
    assert got[0].data_ptr() == out[0].data_ptr() and torch.equal(out[0][:33], rid)
    assert (out[0][33:] == -5).all() and (out[1][33:] == -5).all()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    i2, w2 = rt(view, stream=s)
    s.synchronize()
    assert torch.equal(i2, rid) and torch.equal(w2, rw)
    assert rt(view[:0])[0].shape == (0, 8)
    for bad in (view.t(), view[:, :100], view.expand(33, 128)[:1].expand(4, 128)):
        with pytest.raises(ValueError):
            rt(bad)
    x = view.contiguous()
    rt(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gi, gw = rt(x)
    x.copy_(randn(33, 128, seed=7))
    g.replay()
    ei, ew = rt(x)
    assert torch.equal(gi, ei) and torch.equal(gw, ew)


# ---- norms -----------------------------------------------------------------------

def norm_ref(r, y, dy, post, gate, act, scale, pre, eps, off):
    """(r', bound), (x, bound) in 64 bits; dy: the error y comes with."""
    def stat(v):
        return 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    z, dz = y, dy
    if post is not None:
        f = stat(y) * (post + off)
        # an error dy of y moves its mean square by at most 2 |y| dy
        rel = ((y.abs() * dy).sum(-1, keepdim=True) / (y * y).sum(-1, keepdim=True).clamp(min=1e-300)).clamp(max=1.0)
        z, dz = y * f, dy * f.abs() + (32 * U + rel) * (y * f).abs()
    if gate is not None:
        a = torch.sigmoid(gate) if act == "sigmoid" else gate
        z, dz = z * a, dz * a.abs() + 8 * U * (z * a).abs()
    ro = r + scale * z
    dr = abs(scale) * (dz + 2 * U * z.abs()) + 2 * U * ro.abs() + 2 * U * r.abs()
    p = 1.0 if pre is None else pre + off
    f = stat(ro) * p
    rel = ((ro.abs() * dr).sum(-1, keepdim=True) / (ro * ro).sum(-1, keepdim=True).clamp(min=1e-300)).clamp(max=1.0)
    x = ro * f
    return (ro, dr), (x, dr * abs(f) + (32 * U + rel) * x.abs())


def d64(t):
    return None if t is None else t.double().cpu()


def check_norm(n, h, rt, yt, post=True, gate="none", act="none", scale=0.5, pre=True, off=0.0, eps=1e-6, pad=0,
               seed=0, amp=1.0):
    from moe_prefetch_b200 import BlockNorm

    def rows(w, dtype, s, a=1.0):
        return (a * randn(n, w + pad, seed=seed + s)).to(dtype)[:, pad // 2:pad // 2 + w]
    r, y = rows(h, rt, 1, 3.0), rows(h, yt, 2, amp)
    po = 1 - off + 0.2 * randn(h, seed=3) if post else None
    pr = 1 - off + 0.2 * randn(h, seed=4) if pre is True else None
    g = {"none": None, "token": rows(1, yt, 5) if not pad else rows(1, yt, 5), "channel": randn(h, seed=6),
         "full": rows(h, yt, 7)}[gate]
    nm = BlockNorm(h, post=po, pre=pr if pre is True else pre, gate_act=act, scale=scale, eps=eps, weight_offset=off)
    keep = r.clone()
    ro, x = nm(r, y, gate=g)
    assert torch.equal(r, keep)
    (wr, br), (wx, bx) = norm_ref(d64(r), d64(y), torch.zeros(()).double(), d64(po), d64(g), act,
                                  float(np.float32(scale)), d64(pr), float(np.float32(eps)), off)
    close(ro, wr, br, "r'")
    assert (x is None) == (pre is None)
    if x is not None:
        close(x, wx, bx, "x")
    # in place: r' over r, x over y
    if x is not None:
        nm(r, y, gate=g, out=(r, y))
        assert torch.equal(r, ro) and torch.equal(y, x)


@pytest.mark.parametrize("rt,yt", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("n,h", [(1, 1), (3, 7), (2, 64), (5, 1000), (1, 2048), (40, 2048), (7, 1537), (2, 8192),
                                 (3, 8200), (2, 16384), (2, 16383)])
def test_norm_shapes(n, h, rt, yt):
    check_norm(n, h, rt, yt, gate="full", act="sigmoid")


@pytest.mark.parametrize("gate,act", [("none", "none"), ("token", "none"), ("token", "sigmoid"), ("channel", "sigmoid"),
                                      ("full", "none")])
@pytest.mark.parametrize("post,pre,off", [(True, True, 1.0), (False, True, 0.0), (True, None, 0.0), (False, None, 0.0),
                                          (True, "unit", 1.0)])
@pytest.mark.parametrize("h,pad", [(256, 0), (256, 16), (256, 3), (255, 0)])
def test_norm_forms(gate, act, post, pre, off, h, pad):
    check_norm(6, h, F32, BF16, post=post, gate=gate, act=act, pre=True if pre is True else pre and True, off=off, pad=pad)
    check_norm(6, h, F32, F32, post=post, gate=gate, act=act, pre=pre, off=off, pad=pad) if pre != "unit" else None


@pytest.mark.parametrize("rt,yt", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("h,pad", [(260, 0), (2052, 0), (254, 0), (2046, 2), (1022, 6), (1028, 4), (2050, 0), (6, 0), (12, 4)])
def test_norm_chunk_widths(h, pad, rt, yt):
    """Widths and row strides of every chunk size (8, 4, 2, 1 values), with
    more rows than CTAs, so that the ring of rows turns."""
    check_norm(1300, h, rt, yt, gate="full", act="sigmoid", pad=pad)
    check_norm(3, h, rt, yt, gate="channel", pad=pad)


@pytest.mark.parametrize("amp", [0.0, 1e-20, 1e18])
def test_norm_extreme_rows(amp):
    """Zero rows, rows whose squares underflow, rows whose squares are large."""
    check_norm(4, 512, F32, F32, amp=amp, gate="token", act="sigmoid")


def test_norm_first_block_and_partial_outputs():
    from moe_prefetch_b200 import BlockNorm
    r = 3 * randn(5, 2048, seed=8)
    w = 1 + 0.2 * randn(2048, seed=9)
    nm = BlockNorm(2048, pre=w)
    ro, x = nm(r)
    assert torch.equal(ro, r)
    (_, _), (wx, bx) = norm_ref(d64(r), torch.zeros(5, 2048).double(), torch.zeros(()).double(), None, None, "none",
                                1.0, d64(w), float(np.float32(1e-6)), 0.0)
    close(x, wx, bx, "x")
    x16 = torch.empty(5, 2048, dtype=BF16, device="cuda")
    nm(r, out=(None, x16))     # fp32 residual, bf16 input of the block, r' not written
    close(x16, wx, bx, "x16")
    ones = BlockNorm(2048, pre=True)(r)[1]
    (_, _), (wx, bx) = norm_ref(d64(r), torch.zeros(5, 2048).double(), torch.zeros(()).double(), None, None, "none",
                                1.0, None, float(np.float32(1e-6)), 0.0)
    close(ones, wx, bx, "unit x")
    assert nm(r[:0])[0].shape == (0, 2048)
    for kw in (dict(gate=r), dict(y=r[:4]), dict(y=r.double()), dict(y=r.t()), dict(out=(r, r)), dict(out=(r, None))):
        with pytest.raises((ValueError, RuntimeError)):
            nm(r, **kw)


@pytest.mark.parametrize("n,k,h", [(1, 8, 2048), (33, 9, 2048), (5, 1, 64), (4, 3, 1537), (3, 2, 1026), (2, 8, 16384)])
@pytest.mark.parametrize("add", [False, True])
def test_combine_norm(n, k, h, add):
    from moe_prefetch_b200 import BlockNorm
    rows, r = randn(n * k, h, seed=10), 3 * randn(n, h, seed=11)
    g = torch.Generator().manual_seed(12)
    pos = torch.randperm(n * k, generator=g).int().view(n, k)
    pos[0, 0] = -1                 # an empty pair
    pos[-1, -1] = n * k            # beyond the rows
    w = torch.softmax(randn(n, k, seed=13), -1)
    a = randn(n, h, seed=14) if add else None
    gate, post, pre = randn(n, 1, seed=15), 1 + 0.2 * randn(h, seed=16), 1 + 0.2 * randn(h, seed=17)
    nm = BlockNorm(h, post=post, pre=pre, gate_act="sigmoid", scale=0.7)
    ro, x = nm.combine(r, rows, pos.cuda(), w, add=a, gate=gate)
    ok = (pos >= 0) & (pos < n * k)
    terms = d64(w)[..., None] * torch.where(ok[..., None], d64(rows)[pos.clamp(0, n * k - 1).long()], 0.0)
    y, mag = terms.sum(1), terms.abs().sum(1)
    if add:
        y, mag = y + d64(a), mag + d64(a).abs()
    (wr, br), (wx, bx) = norm_ref(d64(r), y, (k + 1) * U * mag, d64(post), d64(gate), "sigmoid",
                                  float(np.float32(0.7)), d64(pre), float(np.float32(1e-6)), 0.0)
    close(ro, wr, br, "r'")
    close(x, wx, bx, "x")


def test_norm_graph_and_stream():
    from moe_prefetch_b200 import BlockNorm
    h = 2048
    r, y = randn(9, h, seed=18), randn(9, h, seed=19)
    nm = BlockNorm(h, post=1 + 0.2 * randn(h, seed=20), pre=1 + 0.2 * randn(h, seed=21))
    want = nm(r, y)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = nm(r, y, stream=s)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = nm(r, y)
    y.copy_(randn(9, h, seed=22))
    g.replay()
    want = nm(r, y)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- adapters ----------------------------------------------------------------------

def adapters_ref(x, y, a, b, scale, rank, ids):
    """(out, bound) in 64 bits."""
    x, y, a, b, scale, ids = d64(x), d64(y), d64(a), d64(b), d64(scale), ids.cpu()
    out = y.clone()
    bound = U * y.abs()
    n_in = x.shape[1]
    for t in range(x.shape[0]):
        i = int(ids[t])
        if not 0 <= i < a.shape[0]:
            bound[t] = 0
            continue
        r = a.shape[1] if rank is None else int(rank[i])
        low = a[i, :r] @ x[t]
        dlow = (n_in / 8 + 32) * 2 * U * (a[i, :r].abs() @ x[t].abs())
        d = scale[i] * (b[i, :, :r] @ low)
        mag = scale[i].abs() * (b[i, :, :r].abs() @ low.abs())
        out[t] += d
        bound[t] += (r / 8 + 32) * 2 * U * mag + scale[i].abs() * (b[i, :, :r].abs() @ dlow) + 2 * U * out[t].abs()
    return out, bound


def check_adapters(n, n_in, n_out, na, r, xt, wt, ot, order="mixed", ragged=False, pad=0, seed=0, with_y=True):
    from moe_prefetch_b200 import AdapterSet
    x = randn(n, n_in + pad, seed=seed + 1).to(xt)[:, pad // 2:pad // 2 + n_in]
    y = randn(n, n_out + pad, seed=seed + 2).to(ot)[:, pad // 2:pad // 2 + n_out]
    a = (randn(na, r, n_in, seed=seed + 3) / math.sqrt(n_in)).to(wt)
    b = (randn(na, n_out, r, seed=seed + 4) / math.sqrt(r)).to(wt)
    scale = 0.5 + randn(na, seed=seed + 5).abs()
    g = torch.Generator().manual_seed(seed + 6)
    rank = None
    if ragged:
        rank = torch.randint(0, r + 1, (na,), generator=g).int()
        for i in range(na):     # what lies beyond a rank is never used
            a[i, int(rank[i]):] = math.nan
            b[i, :, int(rank[i]):] = math.nan
    ids = torch.randint(-1, na, (n,), generator=g).int()
    if order == "sorted":
        ids = ids.sort()[0]
    elif order == "one":
        ids = torch.full((n,), na - 1, dtype=torch.int32)
    ids[n // 2] = na + 3 if n > 2 else ids[n // 2]     # outside the set
    ids = ids.cuda()
    st = AdapterSet(a, b, scale=scale, rank=None if rank is None else rank.cuda())
    out = st(x, ids, y if with_y else None, out_dtype=ot)
    assert out.dtype == ot
    want, bound = adapters_ref(x, y if with_y else torch.zeros_like(y), a, b, scale, rank, ids)
    close(out, want, bound, "out")
    if with_y:
        left = y.clone()
        skip = (ids < 0) | (ids >= na)
        st(x, ids, y, out=y)
        assert torch.equal(y, out)
        assert torch.equal(y[skip], left[skip])


TYPES = [(F32, BF16, F32), (F32, F16, F32), (BF16, BF16, BF16), (BF16, BF16, F32), (F16, F16, F16), (F16, F16, F32)]


@pytest.mark.parametrize("xt,wt,ot", TYPES)
@pytest.mark.parametrize("n,n_in,n_out,na,r", [
    (1, 1, 1, 1, 1), (1, 2048, 128, 4, 8), (5, 64, 33, 2, 5), (32, 2048, 2048, 16, 16), (3, 1000, 77, 3, 128),
    (130, 200, 65, 5, 24), (70, 1537, 40, 3, 17), (200, 512, 256, 2, 64), (300, 136, 72, 7, 33)])
def test_adapters(n, n_in, n_out, na, r, xt, wt, ot):
    for order in ("mixed", "sorted"):
        check_adapters(n, n_in, n_out, na, r, xt, wt, ot, order=order)


@pytest.mark.parametrize("n", [1, 31, 64, 129, 500])
@pytest.mark.parametrize("xt,wt,ot", TYPES)
def test_adapters_ragged_ranks_strides(n, xt, wt, ot):
    check_adapters(n, 256, 192, 5, 40, xt, wt, ot, ragged=True)
    check_adapters(n, 256, 192, 5, 40, xt, wt, ot, ragged=True, order="sorted", pad=8)
    check_adapters(n, 264, 96, 5, 16, xt, wt, ot, pad=3)
    check_adapters(n, 256, 192, 5, 40, xt, wt, ot, order="one", with_y=False)


@pytest.mark.parametrize("xt,wt,ot", TYPES)
@pytest.mark.parametrize("n,n_in,n_out,na,r,order", [
    (513, 192, 130, 3, 16, "mixed"), (700, 1000, 72, 4, 64, "sorted"), (1111, 136, 96, 9, 23, "sorted"),
    (640, 256, 64, 2, 128, "mixed"), (4097, 64, 40, 50, 8, "mixed"), (8500, 32, 24, 2000, 8, "mixed")])
def test_adapters_long(n, n_in, n_out, na, r, order, xt, wt, ot):
    """Large tiles, several blocks of the token search, more adapters than fit one scan."""
    check_adapters(n, n_in, n_out, na, r, xt, wt, ot, order=order, ragged=na < 10)


def test_adapters_more_tokens_than_a_launch():
    """A call of more tokens than one launch takes, in place, against the same
    rows in two calls."""
    from moe_prefetch_b200 import AdapterSet
    st = AdapterSet((randn(3, 8, 40, seed=1) / 6).to(BF16), randn(3, 24, 8, seed=2).to(BF16), scale=0.5)
    n, cut = 20001, 8192
    x, y = randn(n, 40, seed=3), randn(n, 24, seed=4)
    ids = torch.randint(-1, 3, (n,), generator=torch.Generator().manual_seed(5)).int().cuda()
    want = torch.cat([st(x[a:b], ids[a:b].clone(), y[a:b]) for a, b in ((0, cut), (cut, 2 * cut), (2 * cut, n))])
    assert torch.equal(st(x, ids, y), want)
    ref, bound = adapters_ref(x[-50:], y[-50:], st.a[:, :, :40], st.b, st.scale, None, ids[-50:])
    close(want[-50:], ref, bound, "out")
    st(x, ids, y, out=y)
    assert torch.equal(y, want)


@pytest.mark.parametrize("xt,wt,ot", TYPES)
@pytest.mark.parametrize("n", [7, 600])
def test_adapters_extreme_values(n, xt, wt, ot):
    """An infinity or NaN stays in its row; rows of very different size keep
    their own precision."""
    from moe_prefetch_b200 import AdapterSet
    a, b = (randn(2, 16, 128, seed=1) / 11).to(wt), (randn(2, 72, 16, seed=2) / 4).to(wt)
    x = randn(n, 128, seed=3)
    x[1] *= 2.0 ** -10
    x[2] *= 2.0 ** 10
    x[3, 5], x[4, 6], x[5] = math.inf, math.nan, 0.0
    x = x.to(xt)
    ids = torch.zeros(n, dtype=torch.int32).cuda()
    scale = torch.tensor([0.5, 2.0]).cuda()
    out = AdapterSet(a, b, scale=scale)(x, ids, out_dtype=ot)
    rows = [t for t in range(n) if t not in (3, 4)]
    want, bound = adapters_ref(x[rows], torch.zeros(len(rows), 72), a, b, scale, None, ids[rows])
    close(out[rows], want, bound, "out")
    assert not torch.isfinite(out[3]).any() and torch.isnan(out[4]).all()


def test_adapters_lists_empty_refusals():
    from moe_prefetch_b200 import AdapterSet
    a = [randn(r, 96, seed=r).to(BF16) for r in (4, 9, 16)]
    b = [randn(50, r, seed=r + 1).to(BF16) for r in (4, 9, 16)]
    st = AdapterSet(a, b, scale=0.25)
    x, ids = randn(6, 96, seed=1), torch.tensor([0, 1, 2, -1, 1, 0], dtype=torch.int32).cuda()
    out = st(x, ids)
    for t in range(6):
        i = int(ids[t])
        want = torch.zeros(50).double() if i < 0 else 0.25 * d64(b[i]) @ (d64(a[i]) @ d64(x[t]))
        assert (out[t].double().cpu() - want).abs().max() <= 1e-4 * max(1.0, float(want.abs().max()))
    assert st(x[:0], ids[:0]).shape == (0, 50)
    for call in (lambda: st(x, ids.long()), lambda: st(x, ids[:5]), lambda: st(x[:, :95], ids), lambda: st(x.double(), ids),
                 lambda: st(x, ids, x), lambda: st(x, ids, out=torch.empty(6, 50, device="cuda").t()),
                 lambda: st(x, ids.cpu()), lambda: st(x.cpu(), ids)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):    # an a and a b of different ranks
        AdapterSet(a, b[::-1])
    from moe_prefetch_b200 import MoeError
    with pytest.raises(MoeError):      # fp16 rows beside bf16 weights
        st(x.half(), ids)


def test_adapters_graph_and_stream():
    from moe_prefetch_b200 import AdapterSet
    st = AdapterSet((randn(4, 16, 512, seed=1) / 20).to(BF16), randn(4, 300, 16, seed=2).to(BF16))
    for n in (3, 300):
        x, y = randn(n, 512, seed=3), randn(n, 300, seed=4)
        ids = torch.randint(-1, 4, (n,), generator=torch.Generator().manual_seed(5)).int().cuda()
        want = st(x, ids, y)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        got = st(x, ids, y, stream=s)
        s.synchronize()
        assert torch.equal(got, want)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = st(x, ids, y)
        x.copy_(randn(n, 512, seed=6))
        ids.copy_(ids.flip(0))
        g.replay()
        assert torch.equal(got, st(x, ids, y))
        assert torch.equal(got, st(x, ids, y))      # the same bits every time


# ---- the block through MoeStack -------------------------------------------------------

H = 2048


@pytest.fixture(scope="module", params=[(128, 768, 0), (256, 512, 1)], ids=["e128", "e256shared"])
def stack(request):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from moe_prefetch_b200 import MoeStack
    E, I, n_shared = request.param
    st = MoeStack(n_layers=2, n_expert=E, n_ff=I, n_shared=n_shared)
    st.synth_resident(seed=41, keep_router=True)
    yield st
    st.close()


def router_logits(st, layer, x):
    """moe_router_run's logits: the order every router kernel uses."""
    import ctypes as C
    n = x.shape[0]
    ids = torch.empty(n, 8, dtype=torch.int32, device="cuda")
    w, lg = torch.empty(n, 8, device="cuda"), torch.empty(n, st.n_expert, device="cuda")
    assert st.lib.moe_router_run(C.c_void_p(st.routers[layer].data_ptr()), C.c_void_p(x.data_ptr()), n, st.n_expert, H,
                                 None, 0, 0.0, 8, C.c_void_p(ids.data_ptr()), C.c_void_p(w.data_ptr()),
                                 C.c_void_p(lg.data_ptr()),
                                 C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    return lg


@pytest.mark.parametrize("n_tok,path", [(1, "gemv"), (3, "gemv"), (40, "gemv"), (70, "gemv"), (40, "gemm"), (130, "auto")])
def test_block_without_extras_is_the_layer(stack, n_tok, path):
    """ids, weights and outputs of layer_forward_path, bit for bit; with a
    norm, the norm of exactly that output."""
    from moe_prefetch_b200 import BlockNorm
    x = randn(n_tok, H, seed=n_tok)
    y, ids, w = stack.layer_forward_path(1, x, path)
    y2, ids2, w2 = stack.block_forward(1, x, path=path)
    assert torch.equal(y, y2) and torch.equal(ids, ids2) and torch.equal(w, w2)
    r = 3 * randn(n_tok, H, seed=2)
    nm = BlockNorm(H, post=1 + 0.2 * randn(H, seed=3), pre=1 + 0.2 * randn(H, seed=4), gate_act="sigmoid", scale=0.5)
    gate = randn(n_tok, 1, seed=5)
    ro, xo, ids3, w3 = stack.block_forward(1, x, r=r, norm=nm, gate=gate, path=path)
    assert torch.equal(ids, ids3) and torch.equal(w, w3)
    er, ex = nm(r, y, gate=gate)
    assert torch.equal(ro, er) and torch.equal(xo, ex)
    r2, x2 = r.clone(), x.clone()
    stack.block_forward(1, x2, r=r2, norm=nm, gate=gate, out=(r2, x2), path=path)     # in place
    assert torch.equal(r2, er) and torch.equal(x2, ex)


RULES = [dict(score="sigmoid", bias=True, n_group=4, topk_group=2, group_top=2, scale=1.5),
         dict(score="softmax", bias=True), dict(score="softmax", renorm=False, n_group=8, topk_group=3),
         dict(score="sigmoid", renorm=False, n_group=1)]


@pytest.mark.parametrize("rule", range(len(RULES)))
@pytest.mark.parametrize("n_tok", [1, 5, 70])
def test_layer_routes_by_its_rule(stack, rule, n_tok):
    from moe_prefetch_b200 import MoeError, Routing
    from moe_prefetch_b200.ep import LibEPOps
    kw = dict(RULES[rule])
    kw["bias"] = 0.05 * randn(stack.n_expert, seed=6) if kw.pop("bias", False) else None
    x = randn(n_tok, H, seed=n_tok + 50)
    lg = router_logits(stack, 0, x)
    rid, rw = route_ref(lg, 8, **kw)
    base = stack.layer_forward(0, x)
    stack.set_routing(0, Routing(stack.n_expert, 8, **kw))
    try:
        y, ids, w = stack.layer_forward(0, x)
        assert torch.equal(ids.long().cpu(), rid)
        close(w, rw, 32 * U * rw.abs(), "w")
        b = stack.block_forward(0, x, path="gemv")
        assert torch.equal(b[0], y) and torch.equal(b[1], ids) and torch.equal(b[2], w)
        si, sw = Routing(stack.n_expert, 8, **kw)(lg)
        assert torch.equal(si, ids) and torch.equal(sw, w)
        ei, ew = LibEPOps(stack).route_pack(0, x, 1)[:2]
        assert torch.equal(ei, ids) and torch.equal(ew, w)
        if not stack.n_shared:
            yn, idn, wn = torch.empty_like(x), torch.empty_like(ids), torch.empty_like(w)
            stack.layer_forward_noalloc(0, x, yn, idn, wn)
            assert torch.equal(yn, y) and torch.equal(idn, ids) and torch.equal(wn, w)
        with pytest.raises(MoeError, match="routing rule"):
            stack.decode(x)
        other = stack.layer_forward(1, x)     # the other layer keeps the default
    finally:
        stack.set_routing(0, None)
    again = stack.layer_forward(0, x)
    assert all(torch.equal(p, q) for p, q in zip(base, again))
    assert torch.equal(other[1], stack.layer_forward(1, x)[1])
    stack.decode(x)
    stack.sync()


@pytest.mark.parametrize("n_tok", [1, 6, 200])
def test_block_with_adapters(stack, n_tok):
    """Router adapters on the logits, layer adapters on the output, and the
    norm: each step equal to its operator called alone."""
    from moe_prefetch_b200 import AdapterSet, BlockNorm, Routing
    E = stack.n_expert
    x, r = randn(n_tok, H, seed=70), 3 * randn(n_tok, H, seed=71)
    ids = torch.randint(-1, 3, (n_tok,), generator=torch.Generator().manual_seed(7)).int().cuda()
    ra = AdapterSet((randn(3, 8, H, seed=72) / 45).to(BF16), randn(3, E, 8, seed=73).to(BF16), scale=0.3)
    la = AdapterSet((randn(3, 16, H, seed=74) / 45).to(F16), randn(3, H, 16, seed=75).to(F16), scale=0.3)
    nm = BlockNorm(H, post=1 + 0.2 * randn(H, seed=76), pre=1 + 0.2 * randn(H, seed=77))
    rt = Routing(E, 8, score="sigmoid", bias=0.05 * randn(E, seed=78))
    stack.set_routing(0, rt)
    try:
        lg = ra(x, ids, router_logits(stack, 0, x))
        rid, rw = rt(lg)
        y, i1, w1 = stack.block_forward(0, x, adapter_ids=ids, router_adapters=ra)
        assert torch.equal(i1, rid) and torch.equal(w1, rw)
        y2, i2, w2 = stack.block_forward(0, x, adapter_ids=ids, router_adapters=ra, adapters=la)
        assert torch.equal(i2, rid) and torch.equal(y2, la(x, ids, y))
        ro, xo, i3, w3 = stack.block_forward(0, x, r=r, norm=nm, adapter_ids=ids, router_adapters=ra, adapters=la)
        assert torch.equal(i3, rid)
        # with a norm the adapters' rows are added to the fp32 combine: the same sum
        delta = la(x, ids)
        er, ex = nm(r, y + delta)
        scale = float(er.abs().max())
        assert (ro - er).abs().max() <= 64 * U * scale and (xo - ex).abs().max() <= 64 * U * float(ex.abs().max())
    finally:
        stack.set_routing(0, None)
    # without a rule: softmax over the adapted logits
    _, i4, w4 = stack.block_forward(0, x, adapter_ids=ids, router_adapters=ra)
    rid, rw = route_ref(lg, 8)
    assert torch.equal(i4.long().cpu(), rid)
    close(w4, rw, 32 * U * rw.abs(), "w")


def test_block_prior_and_observation():
    """A rule under the cache prior: delta on resident experts after the
    groups, and the single token is observed as in layer_forward."""
    from moe_prefetch_b200 import MoeCacheConfig, MoeStack, Routing
    E = 64
    st = MoeStack(n_layers=1, n_expert=E, n_ff=256, cache=MoeCacheConfig(n_slots=E, cache_prior=0.3))
    try:
        st.synth_resident(seed=5, keep_router=True)
        st.place(0, list(range(0, E, 2)) + [-1] * (E // 2), copy=False)
        bias = 0.05 * randn(E, seed=8)
        resident = np.zeros(E)
        resident[::2] = np.float32(0.3)
        # every expert the test routes to must be on the device: odd ones lie in groups left out
        bias[1::2] = -2.0
        kw = dict(score="sigmoid", bias=bias, n_group=4, topk_group=2, group_top=2)
        st.set_routing(0, Routing(E, 8, **kw))
        for t in range(4):
            x = randn(1, H, seed=90 + t)
            rid, rw = route_ref(router_logits(st, 0, x), 8, prior=resident, **kw)
            _, ids, w = st.block_forward(0, x)
            assert torch.equal(ids.long().cpu(), rid)
            close(w, rw, 32 * U * rw.abs(), "w")
        st.sync()
        st.step()
        assert st.stats()["hits"] == 32 and st.stats()["misses"] == 0
    finally:
        st.close()


def test_block_layers_in_a_graph(stack):
    """Two layers chained (r and x in place) and captured: the replay equals
    the eager run on new inputs."""
    from moe_prefetch_b200 import BlockNorm
    n = 12
    nms = [BlockNorm(H, post=1 + 0.2 * randn(H, seed=100 + i), pre=1 + 0.2 * randn(H, seed=110 + i), scale=0.5)
           for i in range(2)]
    first = BlockNorm(H, pre=1 + 0.2 * randn(H, seed=120))

    def run(h):
        r, x = first(h)
        for layer in range(2):
            r, x, _, _ = stack.block_forward(layer, x, r=r, norm=nms[layer])
        return r, x

    h = randn(n, H, seed=121)
    run(h)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run(h)
    h.copy_(randn(n, H, seed=122))
    g.replay()
    want = run(h)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_graphs_share_a_context(stack):
    """Two captured layers of one context, of different sizes, replayed in
    turn with eager calls between: the scratch they share holds nothing from
    one call to the next."""
    from moe_prefetch_b200 import AdapterSet, BlockNorm
    nm = BlockNorm(H, post=1 + 0.2 * randn(H, seed=140), pre=1 + 0.2 * randn(H, seed=141))
    ra = AdapterSet((randn(3, 8, H, seed=142) / 45).to(BF16), randn(3, stack.n_expert, 8, seed=143).to(BF16))
    la = AdapterSet((randn(3, 8, H, seed=144) / 45).to(BF16), randn(3, H, 8, seed=145).to(BF16))
    data, graphs = [], []
    for n in (24, 5):      # the larger one first: it sizes the scratch
        x, r = randn(n, H, seed=n), randn(n, H, seed=n + 1)
        ids = torch.randint(-1, 3, (n,), generator=torch.Generator().manual_seed(n)).int().cuda()
        call = lambda x=x, r=r, ids=ids: stack.block_forward(0, x, r=r, norm=nm, adapter_ids=ids, router_adapters=ra,
                                                             adapters=la, path="gemv")
        call()
        data.append((x, call))
    for x, call in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for turn in range(2):
        for i, (x, call) in enumerate(data):
            x.copy_(randn(*x.shape, seed=150 + 2 * turn + i))
        for i in (1, 0, 1):
            graphs[i][0].replay()
            want = data[i][1]()
            assert all(torch.equal(a, b) for a, b in zip(graphs[i][1], want))


def test_calls_at_the_same_time():
    """Two threads, each on its own stream, call the same objects."""
    import threading
    from moe_prefetch_b200 import AdapterSet, BlockNorm, Routing
    rt = Routing(128, 8, score="sigmoid", bias=0.1 * randn(128, seed=1), n_group=4, topk_group=2, group_top=2)
    nm = BlockNorm(512, post=1 + 0.2 * randn(512, seed=2), pre=True, gate_act="sigmoid")
    st = AdapterSet((randn(4, 16, 512, seed=3) / 20).to(BF16), randn(4, 512, 16, seed=4).to(BF16))
    work, bad = [], []
    for i in range(2):
        n = 40 + 500 * i
        lg, r, y = randn(n, 128, seed=10 + i), randn(n, 512, seed=20 + i), randn(n, 512, seed=30 + i)
        gate = randn(n, 1, seed=40 + i) if i else randn(n, 512, seed=40)
        ids = torch.randint(-1, 4, (n,), generator=torch.Generator().manual_seed(i)).int().cuda()
        work.append((lg, r, y, gate, ids, [*rt(lg), *nm(r, y, gate=gate), st(r, ids, y)]))
    torch.cuda.synchronize()

    def run(i):
        lg, r, y, gate, ids, want = work[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got = [*rt(lg), *nm(r, y, gate=gate), st(r, ids, y)]
            torch.cuda.current_stream().synchronize()
        if not all(torch.equal(a, b) for a, b in zip(got, want)):
            bad.append(i)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_block_refusals(stack):
    from moe_prefetch_b200 import AdapterSet, BlockNorm, MoeError, Routing
    x = randn(4, H, seed=130)
    nm = BlockNorm(H, pre=True)
    ad = AdapterSet(randn(2, 8, H, seed=1).to(BF16), randn(2, 64, 8, seed=2).to(BF16))
    for kw in (dict(r=x), dict(norm=nm), dict(gate=x), dict(r=x[:3], norm=nm), dict(r=x, norm=BlockNorm(64, pre=True)),
               dict(adapters=ad, adapter_ids=torch.zeros(4, dtype=torch.int32, device="cuda")),
               dict(r=x, norm=nm, out=(x, None))):
        with pytest.raises(ValueError):
            stack.block_forward(0, x, **kw)
    with pytest.raises(ValueError):
        stack.block_forward(0, x.half())
    with pytest.raises(MoeError):
        stack.set_routing(0, Routing(32, 8))
    assert stack.block_forward(0, x[:0])[0].shape == (0, H)
