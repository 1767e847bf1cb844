"""Cases for timing and checking the projection and log-probability operators.

linear    y = act(x W + bias) + residual, W8A16 weights (int8 with one fp16 scale per column and group of rows)
gated     y = act(x Wg + bg) * (x Wu + bu), both projections in one pass
logprobs  log probability of one given token per row of logits, the row's entropy and its largest alternatives

`run` computes them in elementary torch operations, or, where `own` is set, with the framework's operators.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _framework():
    path = os.path.join(ROOT, "tiny-llm_b200", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tiny_llm_b200

    return tiny_llm_b200


def _linear(name, rows, k, n, group, act="none", bias=False, residual=False, pad=0):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "group": group, "act": act, "bias": bias,
            "residual": residual, "pad": pad}


def _gated(name, rows, k, n, group, act="silu", bias=False, pad=0):
    return {"name": name, "op": "gated", "rows": rows, "k": k, "n": n, "group": group, "act": act, "bias": bias,
            "pad": pad}


def _logprobs(name, rows, vocab, dtype, top, temperature=1.0, masked=False, pad=0):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top,
            "temperature": temperature, "masked": masked, "pad": pad}


def listed():
    return [
        # a layer's output projection for one new token: the smallest call, where latency counts
        _linear("out projection, 1 token", 1, 4096, 4096, 128, residual=True),
        # the down projection of a decode step over a batch
        _linear("down projection, 32 tokens", 32, 14336, 4096, 128, residual=True),
        # odd sizes: a small model's biased projection over a ragged batch, its activations a slice of wider rows
        _linear("biased projection, 77 tokens", 77, 2000, 5003, 64, act="gelu", bias=True, pad=48),
        # the output projection over a long prompt (or many short ones together)
        _linear("out projection, 8192 tokens", 8192, 4096, 4096, 128, residual=True),
        # the gated feed-forward product for one new token, and for a decode step over a batch
        _gated("gated product, 1 token", 1, 4096, 14336, 128),
        _gated("gated product, 32 tokens", 32, 4096, 14336, 128),
        # odd sizes: a small model, biased, groups of 32
        _gated("gated product, 333 tokens", 333, 1096, 2731, 32, act="gelu_tanh", bias=True),
        # a prompt
        _gated("gated product, 4096 tokens", 4096, 4096, 14336, 128),
        # one new token's log probability with the alternatives a client may ask for
        _logprobs("logprobs, 1 row", 1, 128256, "f16", 20),
        # a decode step over a batch
        _logprobs("logprobs, 32 rows", 32, 128256, "f16", 5, temperature=0.8),
        # odd sizes: fp32 logits with most of the vocabulary masked (constrained decoding)
        _logprobs("logprobs, 100 masked rows", 100, 50257, "f32", 10, masked=True, pad=3),
        # scoring of a prompt, no alternatives but the largest
        _logprobs("logprobs, 2048 rows", 2048, 128256, "f16", 1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "gated", "logprobs"])
    if op == "logprobs":
        rows, vocab = _log_int(rng, 1, 2048), _log_int(rng, 500, 160000)
        dtype = rng.choice(["f16", "bf16", "f32"])
        size = 4 if dtype == "f32" else 2
        rows = max(1, min(rows, 500_000_000 // (vocab * size)))
        c = _logprobs("", rows, vocab, dtype, rng.choice([0, 1, 5, 20, 32]), rng.choice([1.0, 0.7, 1.5]),
                      rng.random() < 0.3, rng.choice([0, 0, 1, 8]))
    else:
        k, n = _log_int(rng, 200, 14336), _log_int(rng, 200, 14336)
        rows = _log_int(rng, 1, 4096)
        limit = 8192 * 4096 * 4096
        rows = max(1, min(rows, limit // (k * n * (2 if op == "gated" else 1))))
        group = rng.choice([32, 64, 128])
        act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
        bias = rng.random() < 0.4
        pad = rng.choice([0, 0, 8, 72])
        if op == "linear":
            c = _linear("", rows, k, n, group, act, bias, rng.random() < 0.5, pad)
        else:
            c = _gated("", rows, k, n, group, act, bias, pad)
    del c["name"]
    return c


def _weight(k, n, group, gen):
    """int8 weights and their scales, the product's entries of the size of a trained model's (0.5 / sqrt(k))."""
    w = (torch.randn(k, n, device="cuda", generator=gen, dtype=torch.float16) * 36.0).round_().clamp_(-127, 127).to(torch.int8)
    s = (torch.rand(-(-k // group), n, device="cuda", generator=gen) + 0.5) * (0.5 / 36.0 / math.sqrt(k))
    return w, s.half()


def _inputs(case, seed):
    """What a call is given, from the seed alone."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rows = case["rows"]
    if case["op"] == "logprobs":
        vocab, dtype = case["vocab"], DTYPES[case["dtype"]]
        stride = vocab + case["pad"]
        # a model's logits: a wide body and some tokens that stand out
        wide = torch.empty(rows, stride, device="cuda", dtype=dtype).normal_(0.0, 2.0, generator=gen)
        part = vocab // 24  # one in each 24th of the vocabulary: no index twice
        hot = torch.randint(0, part, (rows, 24), device="cuda", generator=gen) + torch.arange(24, device="cuda") * part
        wide.scatter_(1, hot, (torch.rand(rows, 24, device="cuda", generator=gen) * 10.0 + 5.0).to(dtype))
        logits = wide[:, :vocab]
        tokens = hot[:, 7].to(torch.int32)
        if case["masked"]:
            # a row's allowed tokens: from one token to three in ten of the vocabulary; the given token need not be one
            keep = torch.rand(rows, 1, device="cuda", generator=gen) ** 4 * 0.3
            gone = torch.rand(rows, vocab, device="cuda", generator=gen) >= keep
            gone.scatter_(1, torch.randint(0, vocab, (rows, 1), device="cuda", generator=gen), False)
            logits.masked_fill_(gone, float("-inf"))
        if rows > 4:
            tokens[rows // 2] = -1  # a padded row
        return {"logits": logits, "tokens": tokens}
    k, n, group = case["k"], case["n"], case["group"]
    stride = -(-(k + case["pad"]) // 8) * 8
    x = torch.randn(rows, stride, device="cuda", generator=gen).half()[:, :k]
    d = {"x": x}
    d["w"], d["s"] = _weight(k, n, group, gen)
    if case["op"] == "gated":
        d["w_up"], d["s_up"] = _weight(k, n, group, gen)
    for b in ("bias", "bias_up")[: (0 if not case["bias"] else 2 if case["op"] == "gated" else 1)]:
        d[b] = (torch.randn(n, device="cuda", generator=gen) * 0.3).half()
    if case.get("residual"):
        d["residual"] = torch.randn(rows, n, device="cuda", generator=gen).half()
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = case
    rows = case["rows"]
    if case["op"] == "logprobs":
        d["logprobs"] = torch.empty(rows, device="cuda")
        d["entropy"] = torch.empty(rows, device="cuda")
        d["top_tokens"] = torch.empty(rows, case["top"], device="cuda", dtype=torch.int32)
        d["top_logprobs"] = torch.empty(rows, case["top"], device="cuda")
        return d
    k, n, group = case["k"], case["n"], case["group"]
    d["y"] = torch.empty(rows, n, device="cuda", dtype=torch.float16)
    if own:  # the weights as a program lays them out once, when it loads them
        T = _framework()
        gated = case["op"] == "gated"
        d["packed"] = torch.empty(T.linear_packed_bytes(k, n, group, gated), device="cuda", dtype=torch.uint8)
        T.pack_linear_weight(d["w"].data_ptr(), d["s"].data_ptr(), k, n, group, d["packed"].data_ptr(),
                             d["w_up"].data_ptr() if gated else 0, d["s_up"].data_ptr() if gated else 0,
                             torch.cuda.current_stream().cuda_stream)
    return d


def _act(name, v):
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _product(x, w, s, group, bias):
    k = w.shape[0]
    v = x.float() @ (w.float() * s.float().repeat_interleave(group, 0)[:k])
    return v if bias is None else v + bias.float()


def _plain_logprobs(d, case):
    x = d["logits"].float()
    m = x.max(1, keepdim=True).values
    z = (x - m) / case["temperature"]
    e = torch.exp(z)
    total = e.sum(1)
    log_total = torch.log(total)
    entropy = log_total - torch.where(e > 0, e * z, torch.zeros_like(e)).sum(1) / total
    t = d["tokens"].long()
    given = z.gather(1, t.clamp(min=0)[:, None])[:, 0] - log_total
    given = torch.where(t < 0, torch.zeros_like(given), given)
    # largest first, equal ones by their index: one whole number that orders like (value, -index)
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * 2**32 - torch.arange(x.shape[1], device=x.device)
    at = key.topk(case["top"], 1).indices
    value = z.gather(1, at) - log_total[:, None]
    at = torch.where(value == float("-inf"), torch.full_like(at, -1), at)
    return {"logprobs": given, "entropy": entropy, "top_tokens": at.to(torch.int32), "top_logprobs": value}


ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _own(d, case):
    T = _framework()
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "logprobs":
        T.token_logprobs(d["logits"].data_ptr(), case["rows"], case["vocab"], d["tokens"].data_ptr(),
                         d["logprobs"].data_ptr(), entropy_ptr=d["entropy"].data_ptr(), top_n=case["top"],
                         top_tokens_ptr=d["top_tokens"].data_ptr(), top_logprobs_ptr=d["top_logprobs"].data_ptr(),
                         dtype={"f16": T.TL_F16, "bf16": T.TL_BF16, "f32": T.TL_F32}[case["dtype"]],
                         row_stride=d["logits"].stride(0), temperature=case["temperature"], stream=stream)
        return {name: d[name] for name in ("logprobs", "entropy", "top_tokens", "top_logprobs")}
    bias = d["bias"].data_ptr() if case["bias"] else 0
    if case["op"] == "gated":
        T.linear_gated(d["x"].data_ptr(), case["rows"], d["packed"].data_ptr(), case["k"], case["n"], case["group"],
                       d["y"].data_ptr(), activation=ACTIVATIONS[case["act"]], bias=bias,
                       bias_up=d["bias_up"].data_ptr() if case["bias"] else 0, x_stride=d["x"].stride(0), stream=stream)
    else:
        T.linear(d["x"].data_ptr(), case["rows"], d["packed"].data_ptr(), case["k"], case["n"], case["group"],
                 d["y"].data_ptr(), activation=ACTIVATIONS[case["act"]], bias=bias,
                 residual=d["residual"].data_ptr() if case["residual"] else 0, x_stride=d["x"].stride(0),
                 stream=stream)
    return d["y"]


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    if case["op"] == "logprobs":
        return _plain_logprobs(state, case)
    v = _act(case["act"], _product(state["x"], state["w"], state["s"], case["group"], state.get("bias")))
    if case["op"] == "gated":
        v = v * _product(state["x"], state["w_up"], state["s_up"], case["group"], state.get("bias_up"))
    elif case["residual"]:
        v = v + state["residual"].float()
    return v.half()


def work(case):
    rows = case["rows"]
    if case["op"] == "logprobs":
        size = 4 if case["dtype"] == "f32" else 2
        # per element a comparison, a subtraction, the exponential and two sums
        return {"bytes": rows * (case["vocab"] * size + 12 + 8 * case["top"]), "flops": 5 * rows * case["vocab"]}
    k, n = case["k"], case["n"]
    mats = 2 if case["op"] == "gated" else 1
    moved = mats * (k * n + 2 * n * -(-k // case["group"]) + (2 * n if case["bias"] else 0)) + 2 * rows * (k + n)
    if case.get("residual"):
        moved += 2 * rows * n
    return {"bytes": moved, "flops": 2 * mats * rows * k * n}


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "logprobs":
        out = {"logprobs": [], "entropy": [], "top_logprobs": []}
        for r in range(0, case["rows"], 256):
            z = d["logits"][r:r + 256].double() / case["temperature"]
            log_p = z - torch.logsumexp(z, 1, keepdim=True)
            t = d["tokens"][r:r + 256].long()
            one = log_p[torch.arange(len(t), device=t.device), t.clamp(min=0)]
            one[t < 0] = 0.0
            out["logprobs"].append(one)
            out["entropy"].append(torch.special.entr(log_p.exp()).sum(1))
            out["top_logprobs"].append(log_p.sort(1, descending=True).values[:, :case["top"]].clone())
        out = {name: torch.cat(parts) for name, parts in out.items()}
        out["top_tokens"] = None
        return out

    def product(w, s, bias):
        parts = []
        for j in range(0, case["n"], 4096):
            total = torch.zeros(case["rows"], min(4096, case["n"] - j), device="cuda", dtype=torch.float64)
            for i in range(s.shape[0]):
                at = slice(i * case["group"], min((i + 1) * case["group"], case["k"]))
                total.addmm_(d["x"][:, at].double(), w[at, j:j + 4096].double() * s[i, j:j + 4096].double())
            parts.append(total)
        total = torch.cat(parts, 1)
        return total if bias is None else total + bias.double()

    v = product(d["w"], d["s"], d.get("bias"))
    F = torch.nn.functional
    v = {"none": lambda t: t, "relu": torch.relu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"),
         "silu": F.silu}[case["act"]](v)
    if case["op"] == "gated":
        v = v * product(d["w_up"], d["s_up"], d.get("bias_up"))
    elif case["residual"]:
        v = v + d["residual"].double()
    return v
