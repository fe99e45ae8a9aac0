"""Cases and plain forms of the 8-bit row operators and the token log probabilities.

  add_rmsnorm_quant   residual add + RMSNorm -> INT8 rows with a scale each
  silu_mul_quant      SwiGLU -> INT8 rows with a scale each
  gemm_w8a8           INT8 rows x INT8 weights, a scale for each token and channel
  token_logprobs      log probability of given tokens, entropy, top alternatives

`run` computes the plain form in elementary torch operations, or, where `own`
is true, makes the calls of the C ABI (ec_op_*) that a user makes.
"""
import math
import os

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
CODE = {"f32": 0, "bf16": 1, "f16": 2}  # EC_T_F32, EC_T_BF16, EC_T_F16
EPS = 1e-5
_engine = None


def _lib():
    """The ctypes binding of libengine_cuda.so (the package directory's name
    is not a Python identifier, so it is loaded by path)."""
    global _engine
    if _engine is None:
        import importlib.util
        path = os.path.join(os.getcwd(), "42-berlin-engine_b200", "engine.py")
        spec = importlib.util.spec_from_file_location("ec_engine", path)
        _engine = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_engine)
    return _engine


def listed():
    return [
        # one token of a decode step, f32 activations as the decode path keeps them
        {"name": "norm_decode_f32", "op": "add_rmsnorm_quant", "type": "f32", "rows": 1, "n": 4096,
         "residual": True},
        # a long prompt at the widest model the benchmark runs
        {"name": "norm_prefill_bf16", "op": "add_rmsnorm_quant", "type": "bf16", "rows": 8192,
         "n": 8192, "residual": True},
        # the first norm of a stack (no residual), an odd width, rows padded to 16 bytes
        {"name": "norm_ragged_f16", "op": "add_rmsnorm_quant", "type": "f16", "rows": 333,
         "n": 5003, "residual": False},
        # a small batch of sequences, one token each
        {"name": "swiglu_batch_f32", "op": "silu_mul_quant", "type": "f32", "rows": 8, "n": 14336},
        # a prompt at the widest feed-forward
        {"name": "swiglu_prefill_bf16", "op": "silu_mul_quant", "type": "bf16", "rows": 4096,
         "n": 28672},
        # one token through the fused QKV projection: latency and weight bandwidth
        {"name": "gemm_decode_f32", "op": "gemm_w8a8", "type": "f32", "rows": 1, "m": 6144,
         "k": 4096},
        # 64 sequences through gate and up together: weight bandwidth
        {"name": "gemm_batch_bf16", "op": "gemm_w8a8", "type": "bf16", "rows": 64, "m": 28672,
         "k": 4096},
        # a long prompt through gate and up together: the tensor cores
        {"name": "gemm_prefill_bf16", "op": "gemm_w8a8", "type": "bf16", "rows": 8192, "m": 28672,
         "k": 4096},
        # odd in every size, a long sum
        {"name": "gemm_ragged_f32", "op": "gemm_w8a8", "type": "f32", "rows": 517, "m": 5003,
         "k": 14331},
        # the token a decode step sampled, with its alternatives
        {"name": "logprob_decode_f32", "op": "token_logprobs", "type": "f32", "rows": 1,
         "n": 128256, "top": 5, "temperature": 1.0, "masked": 0.0},
        # the tokens of a prompt scored in one call
        {"name": "logprob_prompt_f32", "op": "token_logprobs", "type": "f32", "rows": 2048,
         "n": 128256, "top": 20, "temperature": 0.7, "masked": 0.0},
        # 16-bit logits (many ties), an odd vocabulary, most tokens barred by a grammar
        {"name": "logprob_masked_bf16", "op": "token_logprobs", "type": "bf16", "rows": 300,
         "n": 32003, "top": 8, "temperature": 1.0, "masked": 0.9},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["add_rmsnorm_quant", "silu_mul_quant", "gemm_w8a8", "gemm_w8a8",
                     "token_logprobs"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "add_rmsnorm_quant":
        n = _log(rng, 64, 16384)
        n = n if rng.random() < 0.4 else -(-n // 64) * 64
        rows = min(_log(rng, 1, 8192), 8192 * 8192 * 2 // (n * SIZE[kind]))
        return {"op": op, "type": kind, "rows": rows, "n": n, "residual": rng.random() < 0.7}
    if op == "silu_mul_quant":
        n = _log(rng, 64, 28672)
        n = n if rng.random() < 0.4 else -(-n // 64) * 64
        rows = min(_log(rng, 1, 8192), 4096 * 28672 * 2 // (n * SIZE[kind]))
        return {"op": op, "type": kind, "rows": rows, "n": n}
    if op == "gemm_w8a8":
        m, k = _log(rng, 64, 128256), _log(rng, 64, 28672)
        if rng.random() < 0.6:
            m, k = -(-m // 64) * 64, -(-k // 64) * 64
        k = min(k, 128256 * 4096 // m)  # up to the language model head's weights
        rows = min(_log(rng, 1, 8192), max(1, 8192 * 28672 * 4096 // (2 * m * k)),
                   max(1, 8192 * 28672 * 2 // (2 * m * SIZE[kind])))
        return {"op": op, "type": kind, "rows": rows, "m": m, "k": k}
    n = _log(rng, 64, 128256)
    rows = min(_log(rng, 1, 4096), max(1, 2048 * 128256 // n))
    return {"op": op, "type": kind, "rows": rows, "n": n, "top": rng.choice([0, 1, 4, 8, 20, 32]),
            "temperature": rng.choice([0.7, 1.0, 1.3]), "masked": rng.choice([0.0, 0.0, 0.5, 0.97])}


def _pad16(n):
    return -(-n // 16) * 16


def _int8(g, rows, k):
    """Quantised rows: normal values of which the largest is about 127."""
    q = torch.empty(rows, _pad16(k), dtype=torch.int8, device="cuda")
    step = max(1, (1 << 27) // q.shape[1])
    for a in range(0, rows, step):
        part = q[a:a + step]
        part.copy_((torch.randn(part.shape, generator=g, device="cuda") * 30).round_().clamp_(-127, 127))
    return q


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dt, rows = case["op"], TYPES[case["type"]], case["rows"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def new(shape, dtype):
        return torch.empty(shape, dtype=dtype, device="cuda")

    s = dict(case, code=CODE[case["type"]], stream=torch.cuda.current_stream().cuda_stream)
    if op == "add_rmsnorm_quant":
        n = case["n"]
        # a residual stream with a few large channels, as deep layers have
        big = 1 + 20 * (torch.rand(n, generator=g, device="cuda") < 0.003).float()
        s["x"] = (normal(rows, n) * 0.5).to(dt)
        s["r"] = (normal(rows, n) * big).to(dt) if case["residual"] else None
        s["w"] = (1 + 0.2 * normal(n)).to(torch.bfloat16)
        s["h"] = new((rows, n), dt) if case["residual"] else None
        s["q"], s["scale"] = new((rows, _pad16(n)), torch.int8), new(rows, torch.float32)
        s["values"] = new((rows, n), torch.bfloat16)
    elif op == "silu_mul_quant":
        n = case["n"]
        s["gu"] = (normal(rows, 2 * n) * 1.5).to(dt)  # one product's output: gate, then up
        s["q"], s["scale"] = new((rows, _pad16(n)), torch.int8), new(rows, torch.float32)
        s["values"] = new((rows, n), torch.bfloat16)
    elif op == "gemm_w8a8":
        m, k = case["m"], case["k"]
        s["xq"], s["wq"] = _int8(g, rows, k), _int8(g, m, k)
        s["sx"] = torch.rand(rows, generator=g, device="cuda") * 0.05 + 0.01
        s["sw"] = torch.rand(m, generator=g, device="cuda") * 1e-3 + 1e-4
        s["y"] = new((rows, m), dt)
    else:
        n = case["n"]
        l = normal(rows, n) * 2.5
        peak = torch.randint(0, n, (rows, 1), generator=g, device="cuda")
        l.scatter_add_(1, peak, 12 * torch.rand(rows, 1, generator=g, device="cuda"))
        if case["masked"]:
            l.masked_fill_(torch.rand(rows, n, generator=g, device="cuda") < case["masked"], -math.inf)
        s["l"] = l.to(dt)
        # mostly the likely token, else any: a masked one has probability 0
        any_ = torch.randint(0, n, (rows, 1), generator=g, device="cuda")
        pick = torch.where(torch.rand(rows, 1, generator=g, device="cuda") < 0.7, peak, any_)
        s["tokens"] = pick[:, 0].to(torch.int32)
        s["top"] = min(case["top"], n)
        s["logprob"], s["entropy"] = new(rows, torch.float32), new(rows, torch.float32)
        s["ids"] = new((rows, s["top"]), torch.int32)
        s["top_logprob"] = new((rows, s["top"]), torch.float32)
    return s


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _values(s):
    """What the 8-bit rows stand for, in 16 bits (which hold them to 2^-9)."""
    return torch.mul(s["q"][:, :s["n"]], s["scale"][:, None], out=s["values"])


def _run_own(s):
    e = _lib()
    L, op = e.lib(), s["op"]
    if op == "add_rmsnorm_quant":
        n = s["n"]
        e.check(L.ec_op_add_rmsnorm_quant(
            s["code"], _ptr(s["x"]), n, _ptr(s["r"]), n, _ptr(s["h"]), n, _ptr(s["w"]), EPS,
            s["rows"], n, _ptr(s["q"]), s["q"].shape[1], _ptr(s["scale"]), s["stream"]))
        out = {"values": _values(s), "scale": s["scale"]}
        return dict(out, h=s["h"]) if s["h"] is not None else out
    if op == "silu_mul_quant":
        n, gu = s["n"], s["gu"]
        e.check(L.ec_op_silu_mul_quant(
            s["code"], gu.data_ptr(), gu.data_ptr() + n * gu.element_size(), 2 * n, s["rows"], n,
            _ptr(s["q"]), s["q"].shape[1], _ptr(s["scale"]), s["stream"]))
        return {"values": _values(s), "scale": s["scale"]}
    if op == "gemm_w8a8":
        e.check(L.ec_op_gemm_w8a8(
            _ptr(s["xq"]), s["xq"].shape[1], _ptr(s["sx"]), _ptr(s["wq"]), s["wq"].shape[1],
            _ptr(s["sw"]), s["code"], _ptr(s["y"]), s["m"], s["m"], s["k"], s["rows"], None,
            s["stream"]))
        return s["y"]
    top = s["top"]
    e.check(L.ec_op_token_logprobs(
        s["code"], _ptr(s["l"]), s["n"], s["n"], s["rows"], _ptr(s["tokens"]),
        s["temperature"], top, _ptr(s["logprob"]), _ptr(s["entropy"]),
        _ptr(s["ids"]) if top else None, _ptr(s["top_logprob"]) if top else None, s["stream"]))
    return {k: s[k] for k in ("logprob", "entropy", "ids", "top_logprob")}


def _quantise(y):
    """f32 rows in 8 bits against their own largest value: the values and the scales."""
    amax = y.abs().amax(1, keepdim=True)
    q = torch.round(y * (127 / amax))
    scale = amax / 127
    return {"values": (q * scale).to(torch.bfloat16), "scale": scale[:, 0]}


def run(s):
    if own:
        return _run_own(s)
    op, dt = s["op"], TYPES[s["type"]]
    if op == "add_rmsnorm_quant":
        h = s["x"]
        if s["r"] is not None:
            h = (h.float() + s["r"].float()).to(dt)
        f = h.float()
        y = f * torch.rsqrt((f * f).mean(1, keepdim=True) + EPS) * s["w"].float()
        out = _quantise(y)
        return dict(out, h=h) if s["r"] is not None else out
    if op == "silu_mul_quant":
        g, u = s["gu"][:, :s["n"]].float(), s["gu"][:, s["n"]:].float()
        return _quantise(g / (1 + torch.exp(-g)) * u)
    if op == "gemm_w8a8":
        k = s["k"]
        acc = s["xq"][:, :k].float() @ s["wq"][:, :k].float().t()
        return (acc * s["sx"][:, None] * s["sw"]).to(dt)
    l = s["l"].float()
    z = l / s["temperature"]
    top = z.amax(1, keepdim=True)
    d = z - torch.where(top == -math.inf, 0, top)  # a row with every token barred: all -inf
    p = torch.exp(d)
    total = p.sum(1)
    total = torch.where(total == 0, 1, total)
    logz = torch.log(total)
    entropy = logz - (p * torch.where(p > 0, d, 0)).sum(1) / total
    logprob = d.gather(1, s["tokens"].long()[:, None])[:, 0] - logz
    # the top of (logit, -index): one integer key orders both
    bits = torch.where(l == 0, 0.0, l).view(torch.int32).long()
    key = torch.where(bits < 0, -2147483648 - bits, bits) * (1 << 17) + (s["n"] - 1 - torch.arange(s["n"], device=l.device))
    ids = s["n"] - 1 - (torch.topk(key, s["top"], 1).values & ((1 << 17) - 1))
    return {"logprob": logprob, "entropy": entropy, "ids": ids.int(),
            "top_logprob": d.gather(1, ids) - logz[:, None]}


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]

    def quantised(y):
        a = y.abs().max(1).values[:, None]
        return {"values": (y / a * 127).round() * a / 127, "scale": a[:, 0] / 127}

    if op == "add_rmsnorm_quant":
        h = s["x"].double()
        if s["r"] is not None:
            h = h + s["r"].double()
        t = h.to(TYPES[s["type"]]).double()  # the operator norms the sum as it is kept
        out = quantised(t / (t.square().sum(1, keepdim=True) / s["n"] + EPS).sqrt() * s["w"].double())
        return dict(out, h=h) if s["r"] is not None else out
    if op == "silu_mul_quant":
        g, u = s["gu"].double().split(s["n"], 1)
        return quantised(torch.sigmoid(g) * g * u)
    if op == "gemm_w8a8":
        y = torch.empty(s["rows"], s["m"], dtype=torch.float64, device="cuda")
        x = s["xq"][:, :s["k"]].double() * s["sx"].double()[:, None]
        for a in range(0, s["m"], 8192):
            w = s["wq"][a:a + 8192, :s["k"]].double() * s["sw"][a:a + 8192, None].double()
            y[:, a:a + 8192] = x @ w.t()
        return y
    out = {"logprob": [], "entropy": [], "top_logprob": []}
    for a in range(0, s["rows"], 256):
        z = s["l"][a:a + 256].double() / s["temperature"]
        lp = z - torch.logsumexp(z, 1, keepdim=True)
        lp = lp.masked_fill(lp.isnan(), -math.inf)  # every token barred
        p = lp.exp()
        out["logprob"].append(lp.gather(1, s["tokens"][a:a + 256, None].long())[:, 0])
        out["entropy"].append(-(p * lp.masked_fill(p == 0, 0.0)).sum(1))
        out["top_logprob"].append(lp.sort(1, descending=True).values[:, :s["top"]])
    return {k: torch.cat(v) for k, v in out.items()} | {"ids": None}


def work(case):
    e, rows = SIZE[case["type"]], case["rows"]
    if case["op"] == "add_rmsnorm_quant":
        n = case["n"]
        streams = 3 if case["residual"] else 1  # x, residual and sum, or x alone
        return {"bytes": rows * n * (streams * e + 1) + 2 * n + 4 * rows, "flops": 8 * rows * n}
    if case["op"] == "silu_mul_quant":
        n = case["n"]
        return {"bytes": rows * n * (2 * e + 1) + 4 * rows, "flops": 8 * rows * n}
    if case["op"] == "gemm_w8a8":
        m, k = case["m"], case["k"]
        return {"bytes": rows * k + m * k + rows * m * e + 4 * (rows + m), "flops": 2 * rows * m * k}
    n, top = case["n"], min(case["top"], case["n"])
    return {"bytes": rows * (n * e + 12 + 8 * top), "flops": 6 * rows * n}
