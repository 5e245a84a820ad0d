"""``QuantLinear`` against a plain product in 64 bits.

Tolerances. Up to 32 tokens (and for fp32 or unaligned x) products are exact, so an output is off by the fp32 sums and its
own rounding: each of about K / 32 + 64 additions by at most 2^-23 (the tensor cores may truncate) of the sum of
magnitudes A = sum |x| (|code scale| + |minimum|), and half a step of the result. Above, each weight is rounded to fp16
(2^-11 of |w|; Q4_K's scale and minimum before that, 2^-11 of each), so at most 2^-10 A more; over many outputs the
roundings average, so their 2-norm is held to 2^-10 of the result's besides."""

import numpy as np
import pytest

from tests.dense_helpers import EPS, TYPES, act, parts, random_rows, torch_dtype, values

pytestmark = pytest.mark.gpu


def reference(qtype, raw, x, K):
    """(y, A) in float64 on the GPU."""
    import torch
    w = torch.from_numpy(values(qtype, raw, K)).cuda()
    p = torch.from_numpy(parts(qtype, raw, K)).cuda()
    return x.double() @ w.T, x.double().abs() @ p.T


def check(y, want, A, K, dtype, prompt):
    import torch
    eps = EPS[dtype]
    err = (y.double() - want).abs()
    tol = (K / 32 + 64) * 2.0 ** -23 * A + (2.0 ** -10 * A if prompt else 0) + (eps / 2) * 1.01 * want.abs() + 2.0 ** -24 * (dtype == "f16")
    assert torch.isfinite(y).all()
    assert (err <= tol).all(), f"max excess {(err - tol).max()}, at {(err - tol).argmax()}"
    rms = err.norm() / want.norm().clamp_min(1e-300)
    assert rms <= eps / 2 + (2.0 ** -10 if prompt else 2.0 ** -19), f"2-norm {rms}"


def make(seed, qtype, dtype, T, K, N, gated=False, activation="silu", ldx=None):
    import torch
    from artlite_b200.linear import QuantLinear
    rng = np.random.default_rng(seed)
    raws = [random_rows(rng, qtype, N, K) for _ in range(2 if gated else 1)]
    x = torch.from_numpy(rng.standard_normal((T, ldx or K)).astype(np.float32)).to(torch_dtype(dtype)).cuda()
    lin = QuantLinear(raws[0], n_in=K, n_out=N, qtype=qtype, act_dtype=dtype, up=raws[1] if gated else None,
                      activation=activation)
    return lin, raws, x


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("qtype", list(TYPES))
@pytest.mark.parametrize("T,K,N", [(1, 256, 16), (1, 512, 1), (3, 768, 37), (8, 2048, 130), (9, 512, 64), (16, 1280, 33),
                                   (17, 256, 48), (32, 2304, 100), (33, 512, 300), (64, 2048, 129), (255, 768, 256),
                                   (257, 256, 640)])
def test_linear(qtype, dtype, T, K, N):
    import torch
    lin, (raw,), x = make(T * 7 + N, qtype, dtype, T, K, N)
    y = torch.full((T + 2, N), 7.0, dtype=x.dtype, device="cuda")
    lin.forward_ptr(x, y, T)
    want, A = reference(qtype, raw, x, K)
    check(y[:T], want, A, K, dtype, T > 32 and dtype != "f32")
    assert (y[T:] == 7).all()
    again = torch.empty_like(y[:T])
    lin.forward_ptr(x, again, T)
    assert torch.equal(again, y[:T])  # (bit-identical repeats)


@pytest.mark.parametrize("qtype", ["Q4_0", "Q4_1", "IQ4_NL"])
@pytest.mark.parametrize("K", [32, 64, 96, 224, 288, 992])
@pytest.mark.parametrize("T", [1, 40])
def test_linear_ragged_rows(qtype, K, T):
    import torch
    lin, (raw,), x = make(K + T, qtype, "bf16", T, K, 70)
    y = torch.empty(T, 70, dtype=x.dtype, device="cuda")
    lin.forward_ptr(x, y, T)
    want, A = reference(qtype, raw, x, K)
    check(y, want, A, K, "bf16", T > 32)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T", [2, 40])
@pytest.mark.parametrize("ldx,ldy,off", [(520, 72, 0), (513, 71, 0), (512, 67, 1), (640, 64, 3), (1024, 200, 8)])
def test_linear_strides_and_offsets(dtype, T, ldx, ldy, off):
    """Row distances and offsets that no 16-byte load takes; the values between rows of y stay."""
    import torch
    K, N = 512, 64
    lin, (raw,), wide = make(T + ldx, "Q4_K", dtype, T + 1, K, N, ldx=ldx)
    flat = wide.reshape(-1)[off:]
    x = torch.as_strided(flat, (T, K), (ldx, 1))
    buf = torch.full((T * ldy + 8,), 5.0, dtype=wide.dtype, device="cuda")
    y = torch.as_strided(buf[off:], (T, N), (ldy, 1))
    before = buf.clone()
    lin.forward_ptr(x, y, T, ldx=ldx, ldy=ldy)
    want, A = reference("Q4_K", raw, x, K)
    check(y, want, A, K, dtype, T > 32 and dtype != "f32")
    torch.as_strided(before[off:], (T, N), (ldy, 1)).copy_(y)
    assert torch.equal(before, buf)


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("qtype", list(TYPES))
@pytest.mark.parametrize("T,K,N", [(1, 512, 33), (12, 768, 128), (32, 256, 20), (50, 512, 200), (300, 1024, 136)])
def test_gated(qtype, dtype, activation, T, K, N):
    """act(g) u: off by |act'| dg |u| + |act(g)| du for its products' errors dg, du (|act'| <= 1.13), the activation's
    own 2^-19, and half a step."""
    import torch
    lin, raws, x = make(N + T, qtype, dtype, T, K, N, gated=True, activation=activation)
    y = torch.empty(T, N, dtype=x.dtype, device="cuda")
    lin.forward_ptr(x, y, T)
    (g, Ag), (u, Au) = (reference(qtype, r, x, K) for r in raws)
    prompt = T > 32 and dtype != "f32"
    rel = (K / 32 + 64) * 2.0 ** -23 + (2.0 ** -10 if prompt else 0)
    a = act(activation, g)
    want = a * u
    dg, du = rel * Ag, rel * Au
    fast = 2.0 ** -21 if dtype == "f32" else 2.0 ** -17
    tol = 1.13 * dg * u.abs() + a.abs() * du + 1.13 * dg * du + (EPS[dtype] / 2 * 1.01 + fast) * want.abs() + 2.0 ** -22 * (dtype == "f16") + 1e-30
    err = (y.double() - want).abs()
    assert (err <= tol).all(), f"max excess {(err - tol).max()}"
    rms = err.norm() / want.norm()
    assert rms <= EPS[dtype] / 2 + (2.0 ** -9 if prompt else 2.0 ** -17), f"2-norm {rms}"


def test_no_tokens_and_host_arrays():
    from artlite_b200.linear import QuantLinear
    rng = np.random.default_rng(5)
    raw = random_rows(rng, "Q4_0", 40, 256)
    lin = QuantLinear(raw, n_in=256, n_out=40, qtype="Q4_0", act_dtype="f32")
    assert lin.forward(np.zeros((0, 256), np.float32)).shape == (0, 40)
    x = rng.standard_normal((5, 256)).astype(np.float32)
    y = lin.forward(x)
    w, p = values("Q4_0", raw, 256), parts("Q4_0", raw, 256)
    want = x.astype(np.float64) @ w.T
    tol = 72 * 2.0 ** -23 * (np.abs(x).astype(np.float64) @ p.T) + 2.0 ** -24 * np.abs(want)
    assert (np.abs(y - want) <= tol).all()


def test_weights_from_device_memory_and_many_tokens_fp32():
    import torch
    from artlite_b200.linear import QuantLinear
    rng = np.random.default_rng(6)
    raw = random_rows(rng, "Q4_K", 48, 512)
    lin = QuantLinear(torch.from_numpy(raw).cuda(), n_in=512, n_out=48, qtype="Q4_K", act_dtype="f32")
    x = torch.from_numpy(rng.standard_normal((777, 512)).astype(np.float32)).cuda()
    y = torch.empty(777, 48, device="cuda")
    lin.forward_ptr(x, y, 777)
    want, A = reference("Q4_K", raw, x, 512)
    check(y, want, A, 512, "f32", False)


@pytest.mark.parametrize("T", [4, 64])
def test_a_token_with_nan_or_infinity_leaves_the_others(T):
    import torch
    lin, (raw,), x = make(11, "Q4_0", "bf16", T, 512, 96)
    x[1, 100] = float("nan")
    x[2, 511] = float("inf")
    y = torch.empty(T, 96, dtype=x.dtype, device="cuda")
    lin.forward_ptr(x, y, T)
    assert torch.isnan(y[1]).all()
    w = torch.from_numpy(values("Q4_0", raw, 512)).cuda()
    assert not torch.isfinite(y[2][w[:, 511] != 0]).any()
    keep = [t for t in range(T) if t not in (1, 2)]
    want, A = reference("Q4_0", raw, x[keep], 512)
    check(y[keep], want, A, 512, "bf16", T > 32)


@pytest.mark.parametrize("T", [4, 64])
@pytest.mark.parametrize("size", [2.0 ** 100, 2.0 ** -100, 2.0 ** 17])
def test_rows_of_any_magnitude(T, size):
    """bf16 rows far outside fp16's range, each row another magnitude."""
    import torch
    lin, (raw,), x = make(12, "Q4_1", "bf16", T, 512, 96)
    s = torch.ones(T, 1, device="cuda")
    s[::2] = size
    x = (x.float() * s).bfloat16()
    y = torch.empty(T, 96, dtype=x.dtype, device="cuda")
    lin.forward_ptr(x, y, T)
    want, A = reference("Q4_1", raw, x, 512)
    check((y.double() / s).float(), want / s, A / s, 512, "bf16", T > 32)


@pytest.mark.parametrize("scale", [2.0 ** -14, 4000.0])
def test_scales_at_the_ends_of_fp16(scale):
    """Blocks whose fp16 scales are subnormal or near the largest."""
    import torch
    from artlite_b200.linear import QuantLinear
    rng = np.random.default_rng(13)
    for qtype in TYPES:
        raw = random_rows(rng, qtype, 64, 512, scale=scale)
        lin = QuantLinear(raw, n_in=512, n_out=64, qtype=qtype, act_dtype="bf16")
        x = torch.from_numpy(rng.standard_normal((40, 512)).astype(np.float32)).bfloat16().cuda()
        for T in (5, 40):
            y = torch.empty(T, 64, dtype=x.dtype, device="cuda")
            lin.forward_ptr(x, y, T)
            want, A = reference(qtype, raw, x[:T], 512)
            check(y, want, A, 512, "bf16", T > 32)


def test_zero_weights_and_zero_rows():
    import torch
    from artlite_b200.linear import QuantLinear
    for qtype in TYPES:
        per, size = TYPES[qtype]
        raw = np.zeros((64, 256 // per * size), np.uint8)
        lin = QuantLinear(raw, n_in=256, n_out=64, qtype=qtype)
        for T in (3, 40):
            x = torch.ones(T, 256, dtype=torch.bfloat16, device="cuda")
            x[1] = 0
            y = torch.full((T, 64), 9.0, dtype=torch.bfloat16, device="cuda")
            lin.forward_ptr(x, y, T)
            assert (y == 0).all()


@pytest.mark.parametrize("T", [2, 48])
def test_streams_and_captured_graphs(T):
    """One handle on two streams at once, and in two captured graphs replayed together."""
    import torch
    lin, (raw,), x0 = make(14, "Q4_K", "bf16", T, 1024, 384)
    xs = [x0, x0.flip(0).contiguous() * 2]
    want = []
    for x in xs:
        y = torch.empty(T, 384, dtype=x.dtype, device="cuda")
        lin.forward_ptr(x, y, T)
        want.append(y)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    ys = [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, x, y in zip(streams, xs, ys):
            lin.forward_ptr(x, y, T, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ys, want))
    graphs = []
    for x, y in zip(xs, ys):
        y.zero_()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            lin.forward_ptr(x, y, T, stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ys, want))


def test_refusals_on_device():
    import torch
    from artlite_b200 import Error
    lin, _, x = make(15, "Q4_0", "bf16", 4, 256, 32)
    y = torch.empty(4, 32, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(Error, match="rows of x 255"):
        lin.forward_ptr(x, y, 4, ldx=255)
    with pytest.raises(Error, match="and of y 31"):
        lin.forward_ptr(x, y, 4, ldy=31)
    with pytest.raises(Error, match="T -1"):
        lin.forward_ptr(x, y, -1)
    with pytest.raises(Error, match="null array"):
        lin.forward_ptr(None, y, 4)
    with pytest.raises(Error, match="not aligned"):
        lin.forward_ptr(x.data_ptr() + 1, y, 4)
    with pytest.raises(Error, match="one of x and y is host"):
        lin.forward_ptr(x.cpu().view(torch.int16).numpy(), y, 4)
    with pytest.raises(Error, match="x has shape"):
        lin.forward(np.zeros((4, 255), np.uint16))
    torch.cuda.synchronize()


def test_a_dense_layer_beside_the_block():
    """The products as a model's dense layer runs them: the gated pair, then the down projection, on a decode batch and on
    a prompt, from the same GGUF rows that an expert would hold; against ref.moe_ffn's SwiGLU of one expert."""
    import torch
    from artlite_b200.linear import QuantLinear
    from oracle import moe_np
    rng = np.random.default_rng(16)
    H, F = 512, 768
    gate, up, down = random_rows(rng, "Q4_0", F, H), random_rows(rng, "Q4_0", F, H), random_rows(rng, "Q4_0", H, F)
    pair = QuantLinear(gate, n_in=H, n_out=F, qtype="Q4_0", up=up)
    out = QuantLinear(down, n_in=F, n_out=H, qtype="Q4_0")
    for T in (1, 5, 100):
        x = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).bfloat16().cuda()
        h = torch.empty(T, F, dtype=x.dtype, device="cuda")
        y = torch.empty(T, H, dtype=x.dtype, device="cuda")
        pair.forward_ptr(x, h, T)
        out.forward_ptr(h, y, T)
        w = [values("Q4_0", r, k).astype(np.float32) for r, k in ((gate, H), (up, H), (down, F))]
        want = moe_np.moe_ffn(x.float().cpu().numpy(), np.zeros((T, 1), np.int32), np.ones((T, 1), np.float32),
                              lambda e: tuple(w))
        assert moe_np.rel_max(y.float().cpu().numpy(), want) <= 1e-2
