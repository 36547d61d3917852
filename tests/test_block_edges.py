"""Refusals of the operators around an expert layer that need no GPU, beyond
the first tests of them: outputs that overlap other tensors."""
import ctypes as C
import random

import pytest

torch = pytest.importorskip("torch")
from test_block_ops import ARG, PTR, lib  # noqa: E402

BASE = 1 << 24


@pytest.fixture
def no_gpu():
    """For calls with made-up pointers of which some are accepted: without a
    GPU those end in a CUDA error before anything is launched."""
    if torch.cuda.is_available():
        pytest.skip("made-up pointers must not reach a GPU")


def norm_rc(n=4, h=64, r=None, rt=0, y=None, yt=0, ro=None, x=None, gate=None, gate_kind=0, post=None, pre=None):
    """moe_block_norm with (byte offset, row stride in elements) per tensor."""
    from moe_prefetch_b200._lib import MoeNorm
    at = lambda t: None if t is None else C.c_void_p(BASE + t[0])
    ld = lambda t: h if t is None else t[1]
    nm = MoeNorm(h, gate_kind, 0, 1.0, 1e-6, 0.0, at(post), at(pre), at(gate), ld(gate))
    return lib().moe_block_norm(C.byref(nm), at(r), rt, ld(r), at(y), yt, ld(y), at(ro), ld(ro), at(x), ld(x), n, None)


FAR = 1 << 20
NORMS = dict(
    stride_of_r=dict(r=(0, 64), ro=(0, 72)),
    stride_of_y=dict(r=(FAR, 64), y=(0, 64), ro=(2 * FAR, 64), x=(0, 80)),
    x_is_r_of_another_type=dict(r=(0, 64), yt=1, x=(0, 64)),
    shifted_r=dict(r=(0, 64), ro=(16, 64)),
    shifted_row=dict(r=(0, 64), ro=(256, 64)),
    before_r=dict(r=(512, 64), ro=(0, 64)),
    shifted_y=dict(r=(FAR, 64), y=(0, 64), ro=(2 * FAR, 64), x=(128, 64)),
    outputs_meet=dict(r=(FAR, 64), ro=(0, 64), x=(1020, 64)),
    into_the_columns=dict(r=(0, 128), ro=(252, 128)),
    next_row=dict(r=(0, 128), ro=(384, 128)),
    gate_per_token=dict(r=(FAR, 64), y=(2 * FAR, 64), gate=(0, 1), gate_kind=1, ro=(8, 64)),
    gate_per_channel=dict(r=(FAR, 64), y=(2 * FAR, 64), gate=(0, 64), gate_kind=2, ro=(0, 64)),
    shifted_gate=dict(r=(FAR, 64), y=(2 * FAR, 64), gate=(0, 64), gate_kind=3, ro=(4, 64)),
    post=dict(r=(FAR, 64), y=(2 * FAR, 64), post=(0, 64), ro=(0, 64)),
    pre=dict(r=(FAR, 64), pre=(1000, 64), x=(0, 64)),
    two_strides=dict(r=(0, 100), ro=(300, 70)))


@pytest.mark.parametrize("case", NORMS)
def test_block_norm_refuses_overlaps(case, no_gpu):
    assert norm_rc(**NORMS[case]) == ARG


ACCEPTED = dict(
    r_in_place=dict(r=(0, 72), ro=(0, 72)),
    y_in_place=dict(r=(FAR, 64), y=(0, 64), yt=1, x=(0, 64)),
    x_over_r=dict(r=(0, 64), x=(0, 64)),
    gate_in_place=dict(r=(FAR, 64), y=(2 * FAR, 64), gate=(0, 64), gate_kind=3, ro=(0, 64)),
    beside_r=dict(r=(0, 128), ro=(256, 128)),
    r_of_one_row=dict(n=1, r=(0, 64), ro=(0, 999)),
    between=dict(r=(0, 192), y=(256, 192), ro=(512, 192)),
    behind=dict(r=(0, 64), ro=(1024, 64)))


@pytest.mark.parametrize("case", ACCEPTED)
def test_block_norm_accepts_rows_that_do_not_meet(case, no_gpu):
    assert norm_rc(**ACCEPTED[case]) not in (0, ARG)


def test_overlap_is_exact(no_gpu):
    """Random rows of r and r_out in one buffer against their sets of bytes."""
    rng = random.Random(1)
    met = 0
    for _ in range(3000):
        h, n = rng.choice([1, 2, 3, 8]), rng.randint(1, 6)
        l1 = h + rng.randint(0, 12)
        l2 = l1 if rng.random() < 0.6 else h + rng.randint(0, 12)
        a, b = 4 * rng.randint(0, 60), 4 * rng.randint(0, 60)
        ra, rb = ({o + 4 * l * i + j for i in range(n) for j in range(4 * h)} for o, l in ((a, l1), (b, l2)))
        same = a == b and (l1 == l2 or n == 1)
        want = bool(ra & rb) and not same
        met += want
        assert (norm_rc(n=n, h=h, r=(a, l1), ro=(b, l2)) == ARG) == want, (h, n, a, l1, b, l2)
    assert 300 < met < 2700


MIB = 1 << 20


@pytest.mark.parametrize("kw", [
    dict(r_out=3 * MIB), dict(x=2 * MIB + 64), dict(r_out=5 * MIB + 4), dict(r_out=6 * MIB, x=6 * MIB + 512),
    dict(r_out=1 * MIB + 4), dict(r_out=4 * MIB + 20), dict(r_out=4 * MIB - 1028)])
def test_combine_norm_refuses_overlaps(kw, no_gpu):
    """Four rows of 64 over pos, y_rows, shifted add, the other output, shifted r,
    and the last and first bytes of w (32 bytes from 4 MiB - 8)."""
    from moe_prefetch_b200._lib import MoeNorm
    d = dict(r=1 * MIB, rows=2 * MIB, pos=3 * MIB, w=4 * MIB - 8, add=5 * MIB, r_out=7 * MIB, x=None)
    d.update(kw)
    p = {k: None if v is None else C.c_void_p(v) for k, v in d.items()}
    nm = MoeNorm(64, 0, 0, 1.0, 1e-6, 0.0, None, None, None, 0)
    assert lib().moe_combine_norm(C.byref(nm), p["r"], 64, p["rows"], 64, 8, p["pos"], p["w"], 2, p["add"], p["r_out"], 64,
                                  p["x"], 64, 4, None) == ARG


@pytest.mark.parametrize("kw", [dict(out=(4 << 20) + 16), dict(out=(4 << 20) - 4), dict(out=5 << 20), dict(y=(6 << 20) + 64),
                                dict(out=1 << 20), dict(out=2 << 20), dict(out=(3 << 20) + 4)])
def test_adapters_refuse_overlaps(kw, no_gpu):
    """out on x, on ids, beside itself on y, on the weights and scales."""
    from moe_prefetch_b200._lib import MoeAdapters
    d = dict(a=1 << 20, b=2 << 20, scale=3 << 20, x=4 << 20, ids=5 << 20, y=None, out=6 << 20)
    d.update(kw)
    p = {k: None if v is None else C.c_void_p(v) for k, v in d.items()}
    st = MoeAdapters(p["a"], p["b"], p["scale"], None, 2, 8, 64, 32, 1, 64)
    assert lib().moe_adapters_apply(C.byref(st), p["ids"], p["x"], 1, 64, p["y"], 32, p["out"], 1, 32, 9, None) == ARG


@pytest.mark.parametrize("kw", [dict(ids=(1 << 20) + 64), dict(w=(1 << 20) + 2000), dict(ids=2 << 20, w=(2 << 20) + 16),
                                dict(w=4 << 20)])
def test_route_refuses_overlaps(kw, no_gpu):
    from moe_prefetch_b200._lib import MoeRouteCfg
    d = dict(logits=1 << 20, ids=2 << 20, w=3 << 20, bias=4 << 20)
    d.update(kw)
    p = {k: C.c_void_p(v) for k, v in d.items()}
    cfg = MoeRouteCfg(64, 4, 0, 1, 1, 1, 1, 1.0)
    assert lib().moe_route(C.byref(cfg), p["logits"], 0, 64, 9, p["bias"], p["ids"], p["w"], None) == ARG


SMEM_MAIN = r"""
// Two threads make the first calls of one kernel with different sizes.  The
// smaller one's cudaFuncSetAttribute is held until the larger one's call has
// ended, or for a while where that waits for the smaller one.
#include "moe_smem.h"

#include <chrono>
#include <cstdio>
#include <thread>

static std::atomic<int> limit{0}, small_inside{0}, large_done{0};
extern "C" cudaError_t cudaGetDevice(int *d) { *d = 0; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute, int bytes) {
    if (bytes == 100) {
        small_inside = 1;
        for (int i = 0; i < 300 && !large_done; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
    }
    limit = bytes;
    return cudaSuccess;
}
static moe::SmemAttr attr;
int main() {
    std::thread a([] { attr.need(nullptr, 100); });
    std::thread b([] {
        while (!small_inside) std::this_thread::yield();
        attr.need(nullptr, 150);
        large_done = 1;
    });
    a.join();
    b.join();
    attr.need(nullptr, 150);
    attr.need(nullptr, 120);
    std::printf("%d\n", limit.load());
    return limit >= 150 ? 0 : 1;
}
"""


def test_shared_memory_limit_never_falls(tmp_path):
    """A kernel's limit after first launches of two sizes from two threads
    allows the larger one (the CUDA runtime replaced by two functions)."""
    import os
    import shutil
    import subprocess
    cuda = next((d for d in (os.environ.get("CUDA_HOME"), "/usr/local/cuda")
                 if d and os.path.exists(os.path.join(d, "include", "cuda_runtime_api.h"))), None)
    if cuda is None or shutil.which("g++") is None:
        pytest.skip("no g++ or CUDA headers")
    src, exe = tmp_path / "smem.cpp", tmp_path / "smem"
    src.write_text(SMEM_MAIN)
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moe_prefetch_b200", "csrc")
    subprocess.check_call(["g++", "-std=c++17", "-pthread", "-I", os.path.join(cuda, "include"), "-I", csrc, "-o", str(exe),
                           str(src)])
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_weights_given_other_memory_are_not_dangling():
    """A weight whose tensor is given other memory (as moving a module does)
    keeps the memory that its address was taken from."""
    from moe_prefetch_b200 import BlockNorm, Routing
    post, pre, bias = (torch.nn.Parameter(torch.zeros(64)) for _ in range(3))
    nm, rt = BlockNorm(64, post=post, pre=pre), Routing(64, 4, bias=bias)
    for t in (post, pre, bias):
        t.data = torch.ones(64)
    assert (nm.post.data_ptr(), nm.pre.data_ptr()) == (nm.nm.post, nm.nm.pre) and nm.with_x
    assert rt.bias.data_ptr() == rt.bias_ptr


def test_masked_scores_are_checked():
    from moe_prefetch_b200 import Routing
    from test_block_ops import route_rc
    for score, code in ((0x100, 0), (0x101, 0), (0x102, ARG), (0x200, ARG), (-1, ARG)):
        assert route_rc(score=score, n_tok=0) == code
    assert Routing(64, 4, masked=True).cfg.score == 0x100 and Routing(64, 4, "sigmoid").cfg.score == 1
