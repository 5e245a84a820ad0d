"""The dense products as a program uses them: with the MoE block on one stream, from several threads, captured before any
other call, with rows far apart, and at the ends of the sizes they take."""

import subprocess
import sys
import textwrap
import threading

import numpy as np
import pytest

from tests.conftest import REPO
from tests.dense_helpers import parts, random_rows, values

pytestmark = pytest.mark.gpu


def close(y, x, qtype, raw, K, prompt, dtype_eps=2.0 ** -7):
    """As tests/test_gpu_linear.py's check, for bf16."""
    import torch
    w = torch.from_numpy(values(qtype, raw, K)).cuda()
    want, A = x.double() @ w.T, x.double().abs() @ torch.from_numpy(parts(qtype, raw, K)).cuda().T
    tol = (K / 32 + 64) * 2.0 ** -23 * A + (2.0 ** -10 * A if prompt else 0) + dtype_eps / 2 * 1.01 * want.abs()
    return bool(((y.double() - want).abs() <= tol).all())


def test_with_the_block_on_one_stream():
    """linear -> MoE block -> gated pair -> linear, enqueued without waiting and captured as one graph: bit-identical to
    the same calls with a wait after each."""
    import torch
    from artlite_b200.linear import QuantLinear
    from oracle import moe_np
    from tests import moe_helpers
    T, H, F = 16, 512, 256
    layer, x, _ = moe_np.make_block(7, T, qtype="Q4_K", E=16, H=H, F=F)
    block = moe_helpers.make_block(layer, T, act="bf16", path="auto", top_k=4)
    rng = np.random.default_rng(1)
    proj = QuantLinear(random_rows(rng, "Q4_0", H, H), n_in=H, n_out=H, qtype="Q4_0")
    pair = QuantLinear(random_rows(rng, "Q4_K", F, H), n_in=H, n_out=F, qtype="Q4_K", up=random_rows(rng, "Q4_K", F, H))
    down = QuantLinear(random_rows(rng, "Q4_0", H, F), n_in=F, n_out=H, qtype="Q4_0")
    bufs = [torch.from_numpy(x.view(np.int16)).cuda()] + [
        torch.zeros(T, n, dtype=torch.int16, device="cuda") for n in (H, H, F, H)]
    st = torch.cuda.Stream()

    def chain(stream, wait=False):
        steps = (lambda: proj.forward_ptr(bufs[0], bufs[1], T, stream=stream),
                 lambda: block.forward_ptr(bufs[1], bufs[2], T, stream=stream),
                 lambda: pair.forward_ptr(bufs[2], bufs[3], T, stream=stream),
                 lambda: down.forward_ptr(bufs[3], bufs[4], T, stream=stream))
        for s in steps:
            s()
            if wait:
                torch.cuda.synchronize()

    torch.cuda.synchronize()
    chain(st.cuda_stream, wait=True)
    want = [b.clone() for b in bufs]
    assert want[4].any()
    torch.cuda.synchronize()
    for _ in range(20):
        chain(st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(bufs, want))
    block.close()


def test_threads_share_a_handle():
    import torch
    from artlite_b200.linear import QuantLinear
    rng = np.random.default_rng(2)
    K, N = 768, 200
    raw = random_rows(rng, "Q4_1", N, K)
    lin = QuantLinear(raw, n_in=K, n_out=N, qtype="Q4_1")
    fails = []

    def work(T):
        st = torch.cuda.Stream()
        x = torch.from_numpy(np.random.default_rng(T).standard_normal((T, K)).astype(np.float32)).bfloat16().cuda()
        y = torch.empty(T, N, dtype=x.dtype, device="cuda")
        torch.cuda.synchronize()
        for _ in range(50):
            lin.forward_ptr(x, y, T, stream=st.cuda_stream)
        st.synchronize()
        if not close(y, x, "Q4_1", raw, K, T > 32):
            fails.append(T)

    threads = [threading.Thread(target=work, args=(T,)) for T in (1, 3, 9, 30, 70, 300)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not fails


CAPTURE_FIRST = """
    import numpy as np, torch
    from artlite_b200.linear import QuantLinear
    from artlite_b200 import ffn
    from tests.dense_helpers import random_rows
    rng = np.random.default_rng(0)
    T, H, F = {T}, 256, 128
    lin = QuantLinear(random_rows(rng, "Q4_0", F, H), n_in=H, n_out=F, qtype="Q4_0")
    x = torch.randn(T, H, device="cuda").bfloat16()
    wg, wu, dh = (torch.randn(n, m, device="cuda").bfloat16() * 0.1 for n, m in ((F, H), (F, H), (T, F)))
    y, h = (torch.zeros(T, F, dtype=x.dtype, device="cuda") for _ in "yh")
    g, u = (torch.zeros(T, F, device="cuda") for _ in "gu")
    dx, dwg, dwu = torch.zeros_like(x), torch.zeros_like(wg), torch.zeros_like(wu)
    work = torch.zeros(ffn.gated_ffn_work_bytes(T, F), dtype=torch.uint8, device="cuda")
    def step():
        s = torch.cuda.current_stream().cuda_stream
        lin.forward_ptr(x, y, T, stream=s)
        ffn.gated_ffn(x, wg, wu, h, T=T, n_in=H, n_ffn=F, gate=g, up=u, stream=s)
        ffn.gated_ffn_backward(dh, x, wg, wu, g, u, work, T=T, n_in=H, n_ffn=F, dx=dx, dw_gate=dwg, dw_up=dwu, stream=s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    graph.replay()
    torch.cuda.synchronize()
    outs = [y, h, g, u, dx, dwg, dwu]
    got = [t.clone() for t in outs]
    assert all(t.any() for t in got)
    for t in outs:
        t.zero_()
    step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, outs))
"""


@pytest.mark.parametrize("T", [2, 60])
def test_the_first_calls_may_be_captured(T):
    """A fresh process whose first forward, training step and workspace are inside a capture."""
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(CAPTURE_FIRST.format(T=T))], cwd=REPO, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("T,ld", [(3, 1 << 30), (40, 1 << 26)])
def test_rows_past_32_bits(T, ld):
    """Rows so far apart that their offsets pass 2^31 values."""
    import torch
    from artlite_b200 import ffn
    from artlite_b200.linear import QuantLinear
    rng = np.random.default_rng(3)
    K, N = 256, 72
    raw = random_rows(rng, "Q4_0", N, K)
    lin = QuantLinear(raw, n_in=K, n_out=N, qtype="Q4_0")
    far = torch.empty((T - 1) * ld + 512, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(far, (T, K), (ld, 1))
    y = torch.as_strided(far[K:], (T, N), (ld, 1))
    near = torch.from_numpy(rng.standard_normal((T, K)).astype(np.float32)).bfloat16().cuda()
    x.copy_(near)
    lin.forward_ptr(x, y, T, ldx=ld, ldy=ld)
    assert close(y.contiguous(), near, "Q4_0", raw, K, T > 32)
    wg, wu = ((torch.randn(N, K, device="cuda") * 0.06).bfloat16() for _ in "gu")
    want = torch.empty(T, N, dtype=torch.bfloat16, device="cuda")
    ffn.gated_ffn(near, wg, wu, want, T=T, n_in=K, n_ffn=N)
    ffn.gated_ffn(x, wg, wu, y, T=T, n_in=K, n_ffn=N, ldx=ld, ldh=ld)
    assert torch.equal(y.contiguous(), want)


@pytest.mark.parametrize("qtype,K,N,T", [("Q4_0", 131072, 40, 1), ("Q4_0", 131072, 40, 5), ("Q4_K", 131072, 24, 20),
                                         ("IQ4_NL", 131072, 24, 2), ("Q4_1", 131072, 24, 40), ("Q4_0", 32, 150001, 1),
                                         ("Q4_K", 256, 150001, 9), ("Q4_0", 32, 150001, 40)])
def test_longest_rows_and_many_rows(qtype, K, N, T):
    import torch
    from artlite_b200.linear import QuantLinear
    rng = np.random.default_rng(4)
    raw = random_rows(rng, qtype, N, K)
    x = torch.from_numpy(rng.standard_normal((T, K)).astype(np.float32)).cuda()
    for dtype, eps in ((torch.bfloat16, 2.0 ** -7), (torch.float32, 2.0 ** -23)):
        lin = QuantLinear(raw, n_in=K, n_out=N, qtype=qtype, act_dtype="bf16" if dtype == torch.bfloat16 else "f32")
        xd = x.to(dtype)
        y = torch.empty(T, N, dtype=dtype, device="cuda")
        lin.forward_ptr(xd, y, T)
        assert close(y, xd, qtype, raw, K, T > 32 and dtype == torch.bfloat16, eps)


def test_rows_longer_than_it_takes():
    from artlite_b200 import Error
    from artlite_b200.linear import QuantLinear
    with pytest.raises(Error, match="at most 131072"):
        QuantLinear(np.zeros((1, 131104 // 32 * 18), np.uint8), n_in=131104, n_out=1, qtype="Q4_0")


@pytest.mark.parametrize("T", [6, 50])
def test_the_same_matrix_twice_and_shared_inputs(T):
    """up the same rows as w; and two outputs of one input on two streams."""
    import torch
    from artlite_b200.linear import QuantLinear
    rng = np.random.default_rng(5)
    raw = random_rows(rng, "Q4_K", 96, 512)
    x = torch.from_numpy(rng.standard_normal((T, 512)).astype(np.float32)).bfloat16().cuda()
    pair = QuantLinear(raw, n_in=512, n_out=96, qtype="Q4_K", up=raw, act_dtype="bf16")
    y = torch.empty(T, 96, dtype=x.dtype, device="cuda")
    pair.forward_ptr(x, y, T)
    g = x.double() @ torch.from_numpy(values("Q4_K", raw, 512)).cuda().T
    want = g * torch.sigmoid(g) * g
    assert ((y.double() - want).norm() / want.norm()) <= 2.0 ** -8 + (2.0 ** -9 if T > 32 else 2.0 ** -17)


@pytest.mark.parametrize("T", [5, 60])
def test_forward_at_large_gate_values(T):
    """silu and gelu far out on both sides: h follows g u or vanishes, never NaN."""
    import torch
    from artlite_b200 import ffn
    from tests.dense_helpers import act
    H, F = 64, 64
    x = (torch.randn(T, H, device="cuda") * 300).bfloat16()
    wg, wu = (torch.randn(F, H, device="cuda").bfloat16() for _ in "gu")
    for name in ("silu", "gelu"):
        h = torch.empty(T, F, dtype=x.dtype, device="cuda")
        ffn.gated_ffn(x, wg, wu, h, T=T, n_in=H, n_ffn=F, activation=name)
        g, u = x.double() @ wg.double().T, x.double() @ wu.double().T
        want = act(name, g) * u
        assert torch.isfinite(h).all()
        assert ((h.double() - want).abs() <= 2.0 ** -7 * want.abs() + 1e-3 * u.abs()).all()
