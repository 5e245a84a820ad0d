"""The dense products beside the mixture-of-experts block, as cases to time and compare: a product with a 4-bit GGUF
matrix (``QuantLinear``), the gated pair act(x Wg^T) * (x Wu^T) over 4-bit matrices (``QuantLinear`` with ``up``) and
over plain bf16 / f16 matrices (``gated_ffn``), and a training step of the latter (``gated_ffn_backward``).

Each case has a plain form (elementary torch operations in fp32, rounded once at the end) and a definition in 64 bits
(``exact``). Dimensions: T token rows, K values a row, N output features."""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BLOCK = {"Q4_0": (32, 18), "Q4_1": (32, 20), "Q4_K": (256, 144), "IQ4_NL": (32, 18)}  # values, bytes a block
_IQ4 = (-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113)


def listed():
    return [
        # one decoded token through an attention projection of the 2048-wide model: the smallest call
        {"name": "linear q4_0 token", "op": "linear", "qtype": "Q4_0", "dtype": "bf16", "T": 1, "K": 2048, "N": 2048, "pad": 0},
        # one token through a wide dense projection
        {"name": "linear q4_k token wide", "op": "linear", "qtype": "Q4_K", "dtype": "bf16", "T": 1, "K": 4096, "N": 12288, "pad": 0},
        # a few drafted tokens in fp32 activations, odd sizes, non-linear 4-bit codes
        {"name": "linear iq4_nl ragged f32", "op": "linear", "qtype": "IQ4_NL", "dtype": "f32", "T": 5, "K": 2080, "N": 5003, "pad": 16},
        # a serving batch, x a slice of a wider buffer
        {"name": "linear q4_1 batch f16", "op": "linear", "qtype": "Q4_1", "dtype": "f16", "T": 16, "K": 4096, "N": 8192, "pad": 64},
        # a prompt through a projection
        {"name": "linear q4_0 prompt", "op": "linear", "qtype": "Q4_0", "dtype": "bf16", "T": 4000, "K": 4096, "N": 4096, "pad": 0},
        # one token through a dense layer's gate and up
        {"name": "gated q4_k token", "op": "qgated", "qtype": "Q4_K", "dtype": "bf16", "T": 1, "K": 2048, "N": 8192, "pad": 0, "act": "silu"},
        # a prompt through a dense layer's gate and up
        {"name": "gated q4_k prompt", "op": "qgated", "qtype": "Q4_K", "dtype": "bf16", "T": 2048, "K": 2048, "N": 6144, "pad": 0, "act": "silu"},
        # plain weights: one token (the decode step of a model being tuned)
        {"name": "ffn bf16 token", "op": "ffn", "dtype": "bf16", "T": 1, "K": 2048, "N": 6144, "pad": 0, "act": "silu"},
        # plain weights: ragged sizes, the tanh-form gelu
        {"name": "ffn f16 ragged gelu", "op": "ffn", "dtype": "f16", "T": 777, "K": 1032, "N": 2056, "pad": 8, "act": "gelu"},
        # plain weights: a long prompt
        {"name": "ffn bf16 prompt", "op": "ffn", "dtype": "bf16", "T": 8192, "K": 4096, "N": 8192, "pad": 0, "act": "silu"},
        # a training step of the 2048-wide model's 768-wide feed-forward, a ragged batch
        {"name": "train bf16 narrow", "op": "train", "dtype": "bf16", "T": 1003, "K": 2048, "N": 768, "pad": 0, "act": "silu"},
        # a training step of a dense layer
        {"name": "train bf16 wide", "op": "train", "dtype": "bf16", "T": 8192, "K": 2048, "N": 8192, "pad": 0, "act": "silu"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "qgated", "ffn", "train"])
    c = {"op": op}
    if op in ("linear", "qgated"):
        c["qtype"] = rng.choice(["Q4_0", "Q4_1", "Q4_K", "IQ4_NL"])
        c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
        per = _BLOCK[c["qtype"]][0]
        c["K"] = per * max(1, _log(rng, 256, 8192) // per)
        c["N"] = _log(rng, 64, 12288)
        # (fp32 activations are for decode batches and short prompts)
        c["T"] = _log(rng, 1, 256 if c["dtype"] == "f32" else 4096)
        c["pad"] = 8 * rng.choice([0, 0, 1, 5, 32])
    else:
        c["dtype"] = rng.choice(["bf16", "bf16", "f16"])
        c["K"] = 8 * _log(rng, 32, 512)
        c["N"] = 8 * _log(rng, 32, 1024)
        c["T"] = _log(rng, 1 if op == "ffn" else 64, 8192)
        if op == "train":  # (no more work than the widest listed step)
            c["T"] = min(c["T"], 8192 * 2048 * 8192 // (c["K"] * c["N"]))
        c["pad"] = 8 * rng.choice([0, 0, 1, 5, 32])
    if op != "linear":
        c["act"] = rng.choice(["silu", "silu", "gelu"])
    return c


def work(case):
    T, K, N = case["T"], case["K"], case["N"]
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("linear", "qgated"):
        per, size = _BLOCK[case["qtype"]]
        mats = 2 if case["op"] == "qgated" else 1
        return {"bytes": mats * N * (K // per) * size + T * (K + N) * e, "flops": 2 * mats * T * N * K}
    if case["op"] == "ffn":
        return {"bytes": 2 * N * K * e + T * (K + N) * e, "flops": 4 * T * N * K}
    # (reads x, both matrices and dh; writes h, dx and both matrices' gradients)
    return {"bytes": 4 * N * K * e + 2 * T * (K + N) * e, "flops": 12 * T * N * K}


# ---------------------------------------------------------------- inputs


def _quantise(qtype, w):
    """(N, K) fp32 weights as raw GGUF rows (N, row bytes) uint8: scales from each group's extremes, codes rounded to
    the nearest."""
    N, K = w.shape
    if qtype == "Q4_K":
        b = w.view(N, K // 256, 8, 32)
        lo = (-b.amin(-1)).clamp_min(0)
        sc = (b.amax(-1) + lo).clamp_min(1e-8) / 15
        d = (sc.amax(-1, keepdim=True) / 63).half()
        dm = (lo.amax(-1, keepdim=True) / 63).half()
        s6 = (sc / d.float().clamp_min(1e-8)).round().clamp(1, 63)
        m6 = (lo / dm.float().clamp_min(1e-8)).round().clamp(0, 63)
        q = ((b + (dm.float() * m6)[..., None]) / (d.float() * s6).clamp_min(1e-8)[..., None]).round().clamp(0, 15).to(torch.uint8)
        s6, m6 = s6.to(torch.uint8), m6.to(torch.uint8)
        head = torch.cat([s6[..., :4] | ((s6[..., 4:] >> 4) << 6), m6[..., :4] | ((m6[..., 4:] >> 4) << 6),
                          (s6[..., 4:] & 15) | ((m6[..., 4:] & 15) << 4)], -1)
        qs = (q[:, :, 0::2] | (q[:, :, 1::2] << 4)).reshape(N, K // 256, 128)
        return torch.cat([d.view(torch.uint8), dm.view(torch.uint8), head, qs], -1).reshape(N, -1).contiguous()
    b = w.view(N, K // 32, 32)
    parts = []
    if qtype == "Q4_1":
        lo, hi = b.amin(-1, keepdim=True), b.amax(-1, keepdim=True)
        d, m = ((hi - lo).clamp_min(1e-8) / 15).half(), lo.half()
        q = ((b - m.float()) / d.float().clamp_min(1e-8)).round().clamp(0, 15)
        parts = [d.view(torch.uint8), m.view(torch.uint8)]
    elif qtype == "Q4_0":
        d = (b.abs().amax(-1, keepdim=True).clamp_min(1e-8) / 8).half()
        q = (b / d.float().clamp_min(1e-8)).round().add(8).clamp(0, 15)
        parts = [d.view(torch.uint8)]
    else:
        d = (b.abs().amax(-1, keepdim=True).clamp_min(1e-8) / 127).half()
        table = torch.tensor(_IQ4, dtype=torch.float32, device=w.device)
        q = torch.bucketize(b / d.float().clamp_min(1e-8), (table[1:] + table[:-1]) / 2)
        parts = [d.view(torch.uint8)]
    q = q.to(torch.uint8)
    return torch.cat(parts + [q[..., :16] | (q[..., 16:] << 4)], -1).reshape(N, -1).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    T, K, N, pad = case["T"], case["K"], case["N"], case["pad"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=dev) * std

    s = {"case": case, "x": normal(T, K + pad).to(dt)[:, :K]}  # (normed activations; rows K + pad apart)
    if case["op"] in ("linear", "qgated"):
        names = ("w", "up") if case["op"] == "qgated" else ("w",)
        for n in names:
            s[n] = _quantise(case["qtype"], normal(N, K, std=K ** -0.5))
        s["y"] = torch.empty(T, N, dtype=dt, device=dev)
        if own:
            from artlite_b200.linear import QuantLinear
            s["linear"] = QuantLinear(s["w"], n_in=K, n_out=N, qtype=case["qtype"], act_dtype=case["dtype"], up=s.get("up"),
                                      activation=case.get("act", "silu"))
        return s
    s["wg"], s["wu"] = normal(N, K, std=K ** -0.5).to(dt), normal(N, K, std=K ** -0.5).to(dt)
    s["h"] = torch.empty(T, N, dtype=dt, device=dev)
    if case["op"] == "train":
        s["dh"] = normal(T, N, std=0.1).to(dt)
        s["g"], s["u"] = (torch.empty(T, N, dtype=torch.float32, device=dev) for _ in "gu")
        s["dx"] = torch.empty(T, K, dtype=dt, device=dev)
        s["dwg"], s["dwu"] = torch.empty_like(s["wg"]), torch.empty_like(s["wu"])
        if own:
            from artlite_b200 import ffn
            s["work"] = torch.empty(ffn.gated_ffn_work_bytes(T, N), dtype=torch.uint8, device=dev)
    return s


# ---------------------------------------------------------------- one pass


def _weights(qtype, raw, K):
    """The rows' values in fp32."""
    N = raw.shape[0]
    per, size = _BLOCK[qtype]
    b = raw.view(N, K // per, size)

    def half(i):
        return b[..., i:i + 2].contiguous().view(torch.float16).float()

    if qtype == "Q4_K":
        d, dm, h = half(0), half(2), b[..., 4:16]
        sc = torch.cat([h[..., :4] & 63, (h[..., 8:] & 15) | ((h[..., :4] >> 6) << 4)], -1).float()
        mn = torch.cat([h[..., 4:8] & 63, (h[..., 8:] >> 4) | ((h[..., 4:8] >> 6) << 4)], -1).float()
        qs = b[..., 16:].reshape(N, K // 256, 4, 32)
        q = torch.stack([qs & 15, qs >> 4], 3).reshape(N, K // 256, 8, 32).float()
        return (q * (d * sc)[..., None] - (dm * mn)[..., None]).reshape(N, K)
    head = 4 if qtype == "Q4_1" else 2
    qs = b[..., head:]
    q = torch.cat([qs & 15, qs >> 4], -1)
    if qtype == "Q4_0":
        w = half(0) * (q.float() - 8)
    elif qtype == "Q4_1":
        w = half(0) * q.float() + half(2)
    else:
        w = half(0) * torch.tensor(_IQ4, dtype=torch.float32, device=raw.device)[q.int()]
    return w.reshape(N, K)


def _act(name, z):
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))


def _act_grad(name, z):
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    c = 2 * math.sqrt(2 / math.pi)
    s = 1 / (1 + torch.exp(-c * (z + 0.044715 * z * z * z)))
    return s + z * s * (1 - s) * c * (1 + 3 * 0.044715 * z * z)


def run(state):
    c = state["case"]
    if own:
        return _run_own(state, c)
    x = state["x"].float()
    dt = state["x"].dtype
    if c["op"] == "linear":
        return (x @ _weights(c["qtype"], state["w"], c["K"]).T).to(dt)
    if c["op"] == "qgated":
        g = x @ _weights(c["qtype"], state["w"], c["K"]).T
        return (_act(c["act"], g) * (x @ _weights(c["qtype"], state["up"], c["K"]).T)).to(dt)
    wg, wu = state["wg"].float(), state["wu"].float()
    g, u = x @ wg.T, x @ wu.T
    a = _act(c["act"], g)
    if c["op"] == "ffn":
        return (a * u).to(dt)
    dh = state["dh"].float()
    dg, du = dh * u * _act_grad(c["act"], g), dh * a
    return {"h": (a * u).to(dt), "dx": (dg @ wg + du @ wu).to(dt), "dwg": (dg.T @ x).to(dt), "dwu": (du.T @ x).to(dt)}


def _run_own(s, c):
    T, K, N = c["T"], c["K"], c["N"]
    stream = torch.cuda.current_stream().cuda_stream
    ld = K + c["pad"]
    if c["op"] in ("linear", "qgated"):
        s["linear"].forward_ptr(s["x"], s["y"], T, ldx=ld, stream=stream)
        return s["y"]
    from artlite_b200 import ffn
    kw = {"T": T, "n_in": K, "n_ffn": N, "dtype": c["dtype"], "activation": c["act"], "ldx": ld, "stream": stream}
    if c["op"] == "ffn":
        ffn.gated_ffn(s["x"], s["wg"], s["wu"], s["h"], **kw)
        return s["h"]
    ffn.gated_ffn(s["x"], s["wg"], s["wu"], s["h"], gate=s["g"], up=s["u"], **kw)
    ffn.gated_ffn_backward(s["dh"], s["x"], s["wg"], s["wu"], s["g"], s["u"], s["work"], dx=s["dx"], dw_gate=s["dwg"],
                           dw_up=s["dwu"], **kw)
    return {"h": s["h"], "dx": s["dx"], "dwg": s["dwg"], "dwu": s["dwu"]}


# ---------------------------------------------------------------- the definition in 64 bits


def _values64(qtype, raw, K):
    """Value k of row n, from the format's definition: the block's scale (and minimum) and the value's 4-bit code."""
    per, size = _BLOCK[qtype]
    k = torch.arange(K, device=raw.device)
    start = (k // per) * size

    def byte(offset):  # (N, K): byte start + offset of each value's block
        return raw[:, start + offset].to(torch.int64)

    def half(offset):
        bits = (byte(offset) | (byte(offset + 1) << 8)).to(torch.int32)
        sign = 1.0 - 2.0 * (bits >> 15).double()
        ex, man = (bits >> 10) & 31, (bits & 1023).double()
        return sign * torch.where(ex == 0, man * 2.0 ** -24, (1024 + man) * torch.exp2(ex.double() - 25))

    if qtype == "Q4_K":
        j = (k % 256) // 32
        code = byte(16 + 32 * (j // 2) + k % 32)
        code = torch.where(j % 2 == 1, code >> 4, code & 15)
        low = j < 4
        a, b, c = byte(4 + j % 4), byte(8 + j % 4), byte(12 + j % 4)
        sc = torch.where(low, a & 63, (c & 15) + 16 * (a >> 6))
        mn = torch.where(low, b & 63, (c >> 4) + 16 * (b >> 6))
        return half(0) * sc.double() * code.double() - half(2) * mn.double()
    i = k % 32
    code = byte((4 if qtype == "Q4_1" else 2) + i % 16)
    code = torch.where(i >= 16, code >> 4, code & 15)
    if qtype == "Q4_0":
        return half(0) * (code.double() - 8)
    if qtype == "Q4_1":
        return half(0) * code.double() + half(2)
    levels = torch.tensor(_IQ4, dtype=torch.float64, device=raw.device)
    return half(0) * torch.take(levels, code)


def _rows(n, f):
    return torch.cat([f(i, min(i + 512, n)) for i in range(0, n, 512)], 1)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    K, N = case["K"], case["N"]
    quant = case["op"] in ("linear", "qgated")

    def product(w):  # x . w^T, 512 rows of w at a time
        return _rows(N, lambda a, b: torch.mm(x, (_values64(case["qtype"], w[a:b], K) if quant else w[a:b].double()).t()))

    if case["op"] == "linear":
        return product(s["w"])
    g, u = product(s["w"] if quant else s["wg"]), product(s["up"] if quant else s["wu"])
    if case["act"] == "silu":
        t = torch.sigmoid(g)
        slope = t + g * t * (1 - t)
    else:  # 0.5 g (1 + tanh(r)), r = sqrt(2 / pi) (g + 0.044715 g^3)
        r = torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
        t = 0.5 * (1 + r)
        slope = t + 0.5 * g * (1 - r * r) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)
    h = g * t * u
    if case["op"] != "train":
        return h
    dh = s["dh"].double()
    dg, du = dh * u * slope, dh * g * t
    dx = torch.mm(dg, s["wg"].double()) + torch.mm(du, s["wu"].double())
    return {"h": h, "dx": dx, "dwg": torch.mm(dg.t(), x), "dwu": torch.mm(du.t(), x)}
