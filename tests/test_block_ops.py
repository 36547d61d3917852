"""Refusals of the operators around an expert layer (routing rules, block
norms, adapters): bad arguments are errors before anything is launched, so
these run without a GPU."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

ARG, UNSUPPORTED = -1, -4
PTR = C.c_void_p(1 << 20)   # never read: every call below fails before a launch


def lib():
    from moe_prefetch_b200 import _lib
    return _lib.load()


def route_rc(n_tok=1, ld=None, dtype=0, logits=PTR, **kw):
    from moe_prefetch_b200._lib import MoeRouteCfg
    d = dict(n_expert=64, k=4, score=0, n_group=1, topk_group=1, group_top=1, renorm=1, scale=1.0)
    d.update(kw)
    cfg = MoeRouteCfg(*d.values())
    return lib().moe_route(C.byref(cfg), logits, dtype, d["n_expert"] if ld is None else ld, n_tok, None, PTR, PTR, None)


@pytest.mark.parametrize("kw,code", [
    (dict(n_expert=0), ARG), (dict(k=0), ARG), (dict(k=65), ARG), (dict(score=2), ARG),
    (dict(n_group=5), ARG), (dict(n_group=0), ARG), (dict(n_group=4, topk_group=5), ARG),
    (dict(n_group=16, topk_group=1, k=5), ARG), (dict(group_top=3), ARG), (dict(group_top=0), ARG),
    (dict(n_expert=513), UNSUPPORTED), (dict(k=33), UNSUPPORTED),
    (dict(n_expert=128, n_group=64, topk_group=64), UNSUPPORTED),
    (dict(ld=63), ARG), (dict(dtype=3), ARG), (dict(n_tok=-1), ARG), (dict(logits=None), ARG)])
def test_route_refuses(kw, code):
    assert route_rc(**kw) == code


def test_no_tokens_is_no_work():
    assert route_rc(n_tok=0, logits=None) == 0


def norm_rc(n_tok=1, r=PTR, r_dtype=0, ld_r=64, y=PTR, dtype=0, ld_y=64, r_out=PTR, x=C.c_void_p(2 << 20), ld=64, **kw):
    from moe_prefetch_b200._lib import MoeNorm
    d = dict(n_embd=64, gate_kind=0, gate_act=0, scale=1.0, eps=1e-6, weight_offset=0.0, post=None, pre=None,
             gate=None, ld_gate=0)
    d.update(kw)
    nm = MoeNorm(*d.values())
    return lib().moe_block_norm(C.byref(nm), r, r_dtype, ld_r, y, dtype, ld_y, r_out, ld, x, ld, n_tok, None)


@pytest.mark.parametrize("kw,code", [
    (dict(n_embd=0), ARG), (dict(n_embd=16385, ld_r=16385, ld_y=16385, ld=16385), UNSUPPORTED),
    (dict(gate_kind=4), ARG), (dict(gate_kind=3), ARG), (dict(gate_kind=3, gate=PTR, ld_gate=63), ARG),
    (dict(gate_act=2), ARG), (dict(r=None), ARG), (dict(r_out=None, x=None), ARG), (dict(r_out=PTR, x=PTR), ARG),
    (dict(r_dtype=1, dtype=0), ARG), (dict(r_dtype=2, dtype=1), ARG), (dict(dtype=7), ARG),
    (dict(ld_r=63), ARG), (dict(ld_y=63), ARG), (dict(ld=63), ARG), (dict(y=None, post=PTR), ARG),
    (dict(y=None, gate_kind=2, gate=PTR), ARG), (dict(n_tok=-2), ARG)])
def test_block_norm_refuses(kw, code):
    assert norm_rc(**kw) == code


@pytest.mark.parametrize("kw,code", [(dict(k=0), ARG), (dict(pos=None), ARG), (dict(w=None), ARG), (dict(n_rows=-1), ARG),
                                     (dict(ld_rows=63), ARG), (dict(rows=None), ARG), (dict(r_out=C.c_void_p(5 << 20)), ARG)])
def test_combine_norm_refuses(kw, code):
    from moe_prefetch_b200._lib import MoeNorm
    d = dict(rows=C.c_void_p(5 << 20), ld_rows=64, n_rows=8, pos=PTR, w=PTR, k=2, r_out=PTR)
    d.update(kw)
    nm = MoeNorm(64, 0, 0, 1.0, 1e-6, 0.0, None, None, None, 0)
    assert lib().moe_combine_norm(C.byref(nm), PTR, 64, d["rows"], d["ld_rows"], d["n_rows"], d["pos"], d["w"], d["k"],
                                  None, d["r_out"], 64, None, 64, 1, None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(rank=12), ARG), (dict(rank=0), ARG), (dict(rank=136), UNSUPPORTED), (dict(lda=60), ARG), (dict(lda=68), ARG),
    (dict(n_in=16392, lda=16392, ld_x=16392), UNSUPPORTED), (dict(dtype=0), ARG), (dict(a=None), ARG),
    (dict(a=C.c_void_p(8)), ARG), (dict(scale=None), ARG), (dict(n_adapters=0), ARG), (dict(n_out=0), ARG),
    (dict(x_dtype=2), ARG), (dict(x_dtype=1, out_dtype=2), ARG), (dict(x_dtype=0, out_dtype=1), ARG),
    (dict(ids=None), ARG), (dict(x=None), ARG), (dict(ld_x=63), ARG), (dict(y=C.c_void_p(2 << 20), ld_y=31), ARG), (dict(ld_out=31), ARG),
    (dict(y=PTR, out=PTR, ld_y=40), ARG), (dict(x=C.c_void_p(3 << 20), out=C.c_void_p(3 << 20)), ARG), (dict(n_tok=-1), ARG)])
def test_adapters_refuse(kw, code):
    from moe_prefetch_b200._lib import MoeAdapters
    d = dict(a=PTR, b=PTR, scale=PTR, ranks=None, n_adapters=2, rank=8, n_in=64, n_out=32, dtype=1, lda=64)
    c = dict(ids=PTR, x=C.c_void_p(4 << 20), x_dtype=1, ld_x=64, y=None, ld_y=32, out=PTR, out_dtype=1, ld_out=32, n_tok=1)
    for k, v in kw.items():
        (d if k in d else c)[k] = v
    if d["n_in"] > 64 and "ld_x" not in kw:
        c["ld_x"] = d["n_in"]
    st = MoeAdapters(*d.values())
    assert lib().moe_adapters_apply(C.byref(st), c["ids"], c["x"], c["x_dtype"], c["ld_x"], c["y"], c["ld_y"], c["out"],
                                    c["out_dtype"], c["ld_out"], c["n_tok"], None) == code


def test_context_calls_refuse_no_context():
    from moe_prefetch_b200._lib import MoeBlock
    b = MoeBlock()
    assert lib().moe_block_forward(None, 0, PTR, 1, C.byref(b), PTR, None, None, 0, None) == ARG
    assert lib().moe_set_routing(None, 0, None, None) == ARG


def test_python_refusals():
    from moe_prefetch_b200 import AdapterSet, BlockNorm, MoeError, Routing
    with pytest.raises(ValueError, match="score"):
        Routing(64, 4, score="tanh")
    with pytest.raises(MoeError):
        Routing(64, 65)
    with pytest.raises(ValueError, match="bias"):
        Routing(64, 4, bias=torch.zeros(63))
    rt = Routing(64, 4)
    with pytest.raises(ValueError, match="CUDA"):
        rt(torch.zeros(2, 64))
    with pytest.raises(ValueError, match="logits must be"):
        rt(torch.zeros(2, 63))
    with pytest.raises(ValueError, match="type"):
        rt(torch.zeros(2, 64, dtype=torch.float64))
    with pytest.raises(ValueError, match="activation"):
        BlockNorm(64, gate_act="tanh")
    with pytest.raises(ValueError, match="post"):
        BlockNorm(64, post=torch.ones(63))
    with pytest.raises(MoeError):
        BlockNorm(20000)
    with pytest.raises(ValueError, match="CUDA"):
        BlockNorm(64)(torch.zeros(2, 64))
    a, b = torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(2, 32, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        AdapterSet(a, b)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        AdapterSet(a.float(), b.float())
    with pytest.raises(ValueError, match="must be"):
        AdapterSet(a, b[:, :, :4])
    with pytest.raises(ValueError, match="must be"):
        AdapterSet(a[:0], b[:0])
