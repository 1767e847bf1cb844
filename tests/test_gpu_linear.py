"""tl_linear and tl_linear_gated on the device against the same products in
float64 over the dequantized weights, at the sizes where the tiles, blocks of
K, scale groups and row blocks end inside something.

Tolerance. The result is rounded once to fp16 (half a unit: 2^-11 of the
value, 2^-25 below the normal range). Before that, products of fp16 and int8
numbers are exact in fp32 and their sums carry, per addition, at most one fp32
unit of the running sum (the tensor cores truncate): at most k 2^-23 of
sum |x w s| over a row's k terms, plus the scaling's and the epilogue's few
roundings; activations have a slope of at most 1.13 (gelu) and the given
functions' own errors of a few units of 2^-23. A gated product multiplies two
such numbers."""
import math

import numpy as np
import pytest

import conftest
import tiny_llm_b200 as T

pytestmark = pytest.mark.gpu

U16, U32 = 2.0**-11, 2.0**-23


@pytest.fixture(autouse=True)
def _need_gpu():
    if not conftest.cuda_available():
        pytest.skip("no CUDA device")


def act64(act, v):
    import torch
    F = torch.nn.functional
    return [lambda t: t, torch.relu, F.gelu, lambda t: F.gelu(t, approximate="tanh"), F.silu][act](v)


class Weight:
    """int8 weight and scales on the device, their values in float64."""

    def __init__(self, k, n, group, gen, scale=None):
        import torch
        self.w = torch.randint(-128, 128, (k, n), device="cuda", generator=gen, dtype=torch.int16).to(torch.int8)
        s = torch.rand(-(-k // group), n, device="cuda", generator=gen) + 0.5
        self.s = (s * (scale or 1.0 / (74.0 * math.sqrt(k)))).half()
        self.v = self.w.double() * self.s.double().repeat_interleave(group, 0)[:k]


def pack(k, n, group, a, b=None):
    import torch
    size = T.linear_packed_bytes(k, n, group, b is not None)
    packed = torch.full((size + 64,), 0x5A, device="cuda", dtype=torch.uint8)
    T.pack_linear_weight(a.w.data_ptr(), a.s.data_ptr(), k, n, group, packed.data_ptr(),
                         b.w.data_ptr() if b else 0, b.s.data_ptr() if b else 0)
    torch.cuda.synchronize()
    assert (packed[size:] == 0x5A).all()
    return packed[:size]


def make_x(rows, k, gen, stride=None):
    import torch
    stride = stride or -(-k // 8) * 8
    buf = torch.full((rows, stride), float("nan"), device="cuda", dtype=torch.float16)  # what lies between rows is never read into a result
    buf[:, :k] = torch.randn(rows, k, device="cuda", generator=gen).half()
    return buf


def bounds(x, W, k, slope=1.13):
    """How far sum x W may be off in fp32 sums of products."""
    return slope * (k + 64) * U32 * (x.abs() @ W.abs())


def run_linear(rows, k, n, group, act=0, bias=False, residual=False, seed=0, x_stride=None, y_stride=None,
               res_stride=None, in_place=False):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(1000 + seed)
    W = Weight(k, n, group, gen)
    packed = pack(k, n, group, W)
    xb = make_x(rows, k, gen, x_stride)
    b = torch.randn(n, device="cuda", generator=gen).half() if bias else None
    ys = y_stride or n
    yb = torch.full((rows + 1, ys), 7.0, device="cuda", dtype=torch.float16)
    rs = res_stride or n
    res = torch.randn(rows, rs, device="cuda", generator=gen).half() if residual else None
    if in_place:
        yb[:rows, :n] = res[:, :n]
    kept = res.clone() if residual else None
    T.linear(xb.data_ptr(), rows, packed.data_ptr(), k, n, group, yb.data_ptr(), bias=b.data_ptr() if bias else 0,
             activation=act, residual=(yb if in_place else res).data_ptr() if residual else 0, x_stride=xb.stride(0),
             y_stride=ys, residual_stride=ys if in_place else rs)
    torch.cuda.synchronize()
    got = yb[:rows, :n]
    x = xb[:, :k].double()
    pre = x @ W.v + (b.double() if bias else 0)
    ref = act64(act, pre) + (kept[:, :n].double() if residual else 0)
    tol = bounds(x, W.v, k) + 16 * U32 * (pre.abs() + ref.abs()) + U16 * ref.abs() + 2.0**-25
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), f"worst {((err - tol).max().item())} at {int((err - tol).argmax())}"
    assert (yb[rows] == 7.0).all() and (yb[:rows, n:] == 7.0).all()  # nothing else is written
    return got


ROWS = [1, 2, 8, 9, 16, 17, 31, 32, 33, 64, 65, 100, 128, 192, 193, 257]


@pytest.mark.parametrize("rows", ROWS)
def test_rows(rows):
    run_linear(rows, 512, 320, 128, residual=True, seed=rows)


@pytest.mark.parametrize("rows", [1, 5, 32, 70])
@pytest.mark.parametrize("k,n,group", [
    (1, 1, 128), (7, 3, 32), (8, 64, 64), (31, 65, 32), (33, 129, 32), (64, 127, 64), (65, 128, 64), (127, 63, 128),
    (128, 200, 128), (129, 1, 128), (255, 77, 32), (1000, 333, 128), (1003, 1001, 64), (4096, 64, 128), (5000, 130, 32),
])
def test_odd_sizes(rows, k, n, group):
    run_linear(rows, k, n, group, act=(k + n) % 5, bias=k % 2 == 1, residual=n % 2 == 1, seed=k * 7 + n)


@pytest.mark.parametrize("rows,k,n,group", [(1, 8192, 20000, 128), (8, 4096, 28672, 64), (12, 6000, 20000, 32),
                                            (30, 4096, 28672, 128), (64, 4096, 20000, 64), (150, 2048, 30000, 32),
                                            (700, 1500, 9000, 128), (2000, 700, 3500, 64)])
def test_many_steps(rows, k, n, group):
    """More steps than the rings hold, more tiles than CTAs."""
    run_linear(rows, k, n, group, residual=True, seed=rows)


@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("act", range(5))
@pytest.mark.parametrize("bias", [False, True])
def test_epilogues(rows, act, bias):
    run_linear(rows, 300, 200, 64, act=act, bias=bias, residual=True, seed=act)


@pytest.mark.parametrize("rows", [4, 48])
def test_strides_and_in_place_residual(rows):
    run_linear(rows, 200, 100, 32, residual=True, x_stride=264, y_stride=111, res_stride=103, seed=1)
    run_linear(rows, 200, 100, 32, residual=True, in_place=True, y_stride=105, seed=2)
    run_linear(rows, 200, 104, 32, residual=True, y_stride=112, res_stride=120, seed=3)


@pytest.mark.parametrize("rows", [1, 8, 20, 33, 130, 200])
@pytest.mark.parametrize("k,n,group", [(256, 64, 128), (129, 33, 64), (1000, 77, 32), (2048, 500, 128), (40, 1, 32)])
@pytest.mark.parametrize("act,bias", [(4, False), (2, True)])
def test_gated(rows, k, n, group, act, bias):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(k + n + rows)
    A, B = Weight(k, n, group, gen), Weight(k, n, group, gen)
    packed = pack(k, n, group, A, B)
    xb = make_x(rows, k, gen)
    ba, bb = (torch.randn(n, device="cuda", generator=gen).half() for _ in range(2))
    y = torch.full((rows + 1, n + 3), 7.0, device="cuda", dtype=torch.float16)
    T.linear_gated(xb.data_ptr(), rows, packed.data_ptr(), k, n, group, y.data_ptr(), activation=act,
                   bias=ba.data_ptr() if bias else 0, bias_up=bb.data_ptr() if bias else 0, x_stride=xb.stride(0),
                   y_stride=n + 3)
    torch.cuda.synchronize()
    x = xb[:, :k].double()
    g = x @ A.v + (ba.double() if bias else 0)
    u = x @ B.v + (bb.double() if bias else 0)
    ag = act64(act, g)
    ref = ag * u
    eg = bounds(x, A.v, k) + 16 * U32 * g.abs()
    eu = bounds(x, B.v, k, 1.0) + 2 * U32 * u.abs()
    tol = eg * u.abs() + eu * ag.abs() + eg * eu + 4 * U32 * ref.abs() + U16 * ref.abs() + 2.0**-25
    err = (y[:rows, :n].double() - ref).abs()
    assert (err <= tol).all(), f"worst {((err - tol).max().item())}"
    assert (y[rows] == 7.0).all() and (y[:rows, n:] == 7.0).all()


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_rows_are_independent(rows):
    """NaN and infinities of one row stay in it; a row's result does not
    depend on the rows beside it or on the run."""
    import torch
    k, n, group = 700, 150, 64
    gen = torch.Generator(device="cuda").manual_seed(5)
    W = Weight(k, n, group, gen)
    packed = pack(k, n, group, W)
    x = make_x(rows, k, gen, 704)
    y = torch.empty(3, rows, n, device="cuda", dtype=torch.float16)
    call = lambda xx, i: T.linear(xx.data_ptr(), rows, packed.data_ptr(), k, n, group, y[i].data_ptr(), x_stride=704)  # noqa: E731
    call(x, 0)
    call(x, 1)
    bad = x.clone()
    bad[1, 3] = float("nan")
    bad[2, 699] = float("inf")
    call(bad, 2)
    torch.cuda.synchronize()
    assert torch.equal(y[0].view(torch.int16), y[1].view(torch.int16))
    assert y[2, 1].isnan().all() and not y[2, 2].isfinite().any()
    keep = [r for r in range(rows) if r not in (1, 2)]
    assert torch.equal(y[0, keep], y[2, keep])


def test_overflow_goes_to_infinity():
    import torch
    k, n, group = 256, 64, 128
    gen = torch.Generator(device="cuda").manual_seed(6)
    W = Weight(k, n, group, gen, scale=0.05)
    W.w.fill_(127)
    packed = pack(k, n, group, W)
    x = torch.full((40, k), 100.0, device="cuda", dtype=torch.float16)
    y = torch.empty(40, n, device="cuda", dtype=torch.float16)
    for rows in (2, 40):
        T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y.data_ptr())
        assert (y[:rows] == float("inf")).all()


@pytest.mark.parametrize("rows", [1, 33])
def test_streams_and_graphs(rows):
    """Two calls at once on two streams, and a captured call replayed on new
    activations, give what single calls give."""
    import torch
    k, n, group = 4096, 512, 128
    gen = torch.Generator(device="cuda").manual_seed(7)
    W = Weight(k, n, group, gen)
    packed = pack(k, n, group, W)
    xs = [make_x(rows, k, gen) for _ in range(2)]
    ref = [torch.empty(rows, n, device="cuda", dtype=torch.float16) for _ in range(2)]
    for x, y in zip(xs, ref):
        T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y.data_ptr())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = [torch.empty(20, rows, n, device="cuda", dtype=torch.float16) for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(20):
        for s, x, y in zip(streams, xs, out):
            T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y[i].data_ptr(), stream=s.cuda_stream)
    torch.cuda.synchronize()
    for y, r in zip(out, ref):
        assert all(torch.equal(y[i], r) for i in range(20))
    x, y = xs[0].clone(), torch.empty_like(ref[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y.data_ptr(),
                     stream=torch.cuda.current_stream().cuda_stream)
    for i in (1, 0):
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref[i])


def test_pack_then_product_on_one_stream():
    """The product right behind the packing of its weight, without a wait."""
    import torch
    k, n, group = 2048, 2048, 128
    gen = torch.Generator(device="cuda").manual_seed(8)
    weights = [Weight(k, n, group, gen) for _ in range(4)]
    x = make_x(4, k, gen)
    packed = torch.zeros(T.linear_packed_bytes(k, n, group), device="cuda", dtype=torch.uint8)
    y = torch.empty(4, 4, n, device="cuda", dtype=torch.float16)
    torch.cuda.synchronize()
    for i, W in enumerate(weights):  # one buffer, packed again between the products
        T.pack_linear_weight(W.w.data_ptr(), W.s.data_ptr(), k, n, group, packed.data_ptr())
        T.linear(x.data_ptr(), 4, packed.data_ptr(), k, n, group, y[i].data_ptr())
    torch.cuda.synchronize()
    for i, W in enumerate(weights):
        again = pack(k, n, group, W)
        z = torch.empty(4, n, device="cuda", dtype=torch.float16)
        T.linear(x.data_ptr(), 4, again.data_ptr(), k, n, group, z.data_ptr())
        torch.cuda.synchronize()
        assert torch.equal(y[i], z)


def test_a_layers_end_and_the_head():
    """Output projection with its residual, gated product, down projection
    with its residual, LM head, log probabilities and sampling of the same
    logits, as a decode step runs them: every step against float64 on the
    step's own (fp16) input."""
    import torch
    rows, hidden, inter, vocab, group = 6, 256, 688, 1003, 64
    gen = torch.Generator(device="cuda").manual_seed(9)
    mats = {m: Weight(a, b, group, gen) for m, a, b in
            [("o", hidden, hidden), ("g", hidden, inter), ("u", hidden, inter), ("d", inter, hidden), ("head", hidden, vocab)]}
    po, pd, ph = (pack(*mats[m].w.shape, group, mats[m]) for m in ("o", "d", "head"))
    pg = pack(hidden, inter, group, mats["g"], mats["u"])
    attn, h = make_x(rows, hidden, gen), make_x(rows, hidden, gen)
    h0 = h.clone()
    mid = torch.empty(rows, inter, device="cuda", dtype=torch.float16)
    stride = 1008
    logits = torch.empty(rows, stride, device="cuda", dtype=torch.float16)
    tokens = torch.empty(rows, device="cuda", dtype=torch.int32)
    lp, ent = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    T.linear(attn.data_ptr(), rows, po.data_ptr(), hidden, hidden, group, h.data_ptr(), residual=h.data_ptr())
    torch.cuda.synchronize()
    h1 = h.clone()
    T.linear_gated(h.data_ptr(), rows, pg.data_ptr(), hidden, inter, group, mid.data_ptr())
    T.linear(mid.data_ptr(), rows, pd.data_ptr(), inter, hidden, group, h.data_ptr(), residual=h.data_ptr())
    T.linear(h.data_ptr(), rows, ph.data_ptr(), hidden, vocab, group, logits.data_ptr(), y_stride=stride)
    T.sample_tokens(logits.data_ptr(), stride, rows, vocab, tokens.data_ptr())
    T.token_logprobs(logits.data_ptr(), rows, vocab, tokens.data_ptr(), lp.data_ptr(), ent.data_ptr(), row_stride=stride)
    torch.cuda.synchronize()

    def near(got, ref, tol):
        assert ((got.double() - ref).abs() <= tol + U16 * ref.abs() + 2.0**-25).all()

    near(h1, attn.double() @ mats["o"].v + h0.double(), bounds(attn.double(), mats["o"].v, hidden) + 4 * U32)
    g, u = h1.double() @ mats["g"].v, h1.double() @ mats["u"].v
    e = bounds(h1.double(), mats["g"].v, hidden) + 16 * U32 * g.abs()
    e2 = bounds(h1.double(), mats["u"].v, hidden)
    near(mid, act64(4, g) * u, e * u.abs() + e2 * g.abs() + e * e2)
    near(h, mid.double() @ mats["d"].v + h1.double(), bounds(mid.double(), mats["d"].v, inter) + 4 * U32 * h1.abs().double())
    near(logits[:, :vocab], h.double() @ mats["head"].v, bounds(h.double(), mats["head"].v, hidden))
    logp = torch.log_softmax(logits[:, :vocab].double(), 1)
    assert torch.equal(logits.gather(1, tokens.long()[:, None])[:, 0], logits[:, :vocab].max(1).values)
    assert ((lp.double() - logp.max(1).values).abs() < 4e-6).all()
    assert ((ent.double() + (logp.exp() * logp).sum(1)).abs() < 4e-5).all()
    assert np.isfinite(h.float().cpu().numpy()).all()


@pytest.mark.parametrize("rows", [3, 40, 130])
@pytest.mark.parametrize("gated", [False, True])
def test_unaligned_outputs_and_epilogue_inputs(rows, gated):
    """y, bias and residual on odd elements (2-byte aligned only)."""
    import torch
    k, n, group = 320, 136, 64
    gen = torch.Generator(device="cuda").manual_seed(12)
    A, B = Weight(k, n, group, gen), Weight(k, n, group, gen)
    packed = pack(k, n, group, A, B if gated else None)
    x = make_x(rows, k, gen)
    bias = torch.randn(2, n + 1, device="cuda", generator=gen).half()
    res = torch.randn(rows * (n + 8) + 1, device="cuda", generator=gen).half()
    y = torch.full((rows * (n + 8) + 2,), 7.0, device="cuda", dtype=torch.float16)
    even = torch.empty(rows, n, device="cuda", dtype=torch.float16)  # the same with everything aligned
    b0, b1, r0 = bias[0, 1:].clone(), bias[1, 1:].clone(), res[1:].view(rows, n + 8)[:, :n].clone()
    if gated:
        T.linear_gated(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y[1:].data_ptr(), activation=4,
                       bias=bias[0, 1:].data_ptr(), bias_up=bias[1, 1:].data_ptr(), y_stride=n + 8)
        T.linear_gated(x.data_ptr(), rows, packed.data_ptr(), k, n, group, even.data_ptr(), activation=4,
                       bias=b0.data_ptr(), bias_up=b1.data_ptr())
    else:
        T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y[1:].data_ptr(), activation=2,
                 bias=bias[0, 1:].data_ptr(), residual=res[1:].data_ptr(), y_stride=n + 8, residual_stride=n + 8)
        T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, even.data_ptr(), activation=2,
                 bias=b0.data_ptr(), residual=r0.data_ptr())
    torch.cuda.synchronize()
    got = y[1:-1].view(rows, n + 8)
    assert torch.equal(got[:, :n], even) and (got[:, n:] == 7.0).all() and y[0] == 7.0 and y[-1] == 7.0


@pytest.mark.parametrize("rows", [8, 20, 129])
def test_far_rows(rows):
    """Row offsets past 2^31 elements in the activations, residual and output."""
    import torch
    k, n, group = 136, 72, 128
    stride = ((1 << 31) // (rows - 1) // 8 + 8) * 8
    gen = torch.Generator(device="cuda").manual_seed(13)
    W = Weight(k, n, group, gen)
    packed = pack(k, n, group, W)
    buf = torch.empty(rows * stride, device="cuda", dtype=torch.float16)
    far = buf.view(rows, stride)
    x = make_x(rows, k, gen)
    res = torch.randn(rows, n, device="cuda", generator=gen).half()
    far[:, :k], far[:, 256:256 + n], far[:, 512:512 + n] = x, res, 7.0
    y = torch.empty(rows, n, device="cuda", dtype=torch.float16)
    T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y.data_ptr(), residual=res.data_ptr())
    T.linear(far.data_ptr(), rows, packed.data_ptr(), k, n, group, far[:, 512:].data_ptr(), residual=far[:, 256:].data_ptr(),
             x_stride=stride, y_stride=stride, residual_stride=stride)
    torch.cuda.synchronize()
    assert torch.equal(far[:, 512:512 + n], y)


def test_first_calls_inside_a_capture():
    """A process whose first calls of every kernel are captured."""
    import subprocess
    import sys
    from pathlib import Path
    script = """
import sys, torch
sys.path[:0] = sys.argv[1:]
import tiny_llm_b200 as T
k, n = 512, 192
w = torch.randint(-128, 128, (k, n), device="cuda", dtype=torch.int16).to(torch.int8)
s = torch.rand(4, n, device="cuda").half()
p = torch.empty(T.linear_packed_bytes(k, n, 128), device="cuda", dtype=torch.uint8)
T.pack_linear_weight(w.data_ptr(), s.data_ptr(), k, n, 128, p.data_ptr())
x = torch.randn(300, k, device="cuda").half()
y = torch.zeros(5, 300, n, device="cuda", dtype=torch.float16)
lp = torch.zeros(2, 300, device="cuda")
t = torch.zeros(300, device="cuda", dtype=torch.int32)
torch.cuda.synchronize()
def calls(out, lps, stream):
    for i, rows in enumerate((3, 20, 50, 300)):
        T.linear(x.data_ptr(), rows, p.data_ptr(), k, n, 128, out[i].data_ptr(), stream=stream)
    T.token_logprobs(out[3].data_ptr(), 300, n, t.data_ptr(), lps.data_ptr(), stream=stream)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    calls(y, lp[0], torch.cuda.current_stream().cuda_stream)
g.replay()
torch.cuda.synchronize()
z = torch.zeros_like(y)
calls(z, lp[1], 0)
torch.cuda.synchronize()
assert torch.equal(y, z) and torch.equal(lp[0], lp[1]) and y[:4].abs().amax((1, 2)).min() > 0
"""
    root = Path(T.__file__).resolve().parents[1]
    subprocess.run([sys.executable, "-c", script, str(root)], check=True, timeout=300)


@pytest.mark.parametrize("rows", [4, 33, 130])
def test_logits_written_between_two_readers(rows):
    """log probabilities -> product into the same logits -> log probabilities,
    back to back and replayed: every reader sees the product before it, not
    what an earlier reader loaded."""
    import torch
    k, vocab, group, top, n = 512, 4096, 128, 4, 24
    gen = torch.Generator(device="cuda").manual_seed(rows)
    W = Weight(k, vocab, group, gen)
    packed = pack(k, vocab, group, W)
    xs = [make_x(rows, k, gen) for _ in range(3)]
    tokens = torch.arange(rows, device="cuda", dtype=torch.int32) * 7 % vocab
    logits = torch.empty(rows, vocab, device="cuda", dtype=torch.float16)

    def outputs(m):
        return (torch.empty(m, rows, device="cuda"), torch.empty(m, rows, device="cuda"),
                torch.empty(m, rows, top, device="cuda", dtype=torch.int32),
                torch.empty(m, rows, top, device="cuda"))

    def step(x, out, i, stream):
        T.linear(x.data_ptr(), rows, packed.data_ptr(), k, vocab, group, logits.data_ptr(), stream=stream)
        T.token_logprobs(logits.data_ptr(), rows, vocab, tokens.data_ptr(), out[0][i].data_ptr(), out[1][i].data_ptr(),
                         top, out[2][i].data_ptr(), out[3][i].data_ptr(), stream=stream)

    ref, got = outputs(3), outputs(n)
    for i, x in enumerate(xs):
        step(x, ref, i, 0)
        torch.cuda.synchronize()
    assert not torch.equal(ref[0][0], ref[0][1])
    stream = torch.cuda.Stream()
    for i in range(n):
        step(xs[i % 3], got, i, stream.cuda_stream)
    torch.cuda.synchronize()
    for g, r in zip(got, ref):
        assert all(torch.equal(g[i], r[i % 3]) for i in range(n))
    for g in got:
        g.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(n):
            step(xs[i % 3], got, i, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for g, r in zip(got, ref):
        assert all(torch.equal(g[i], r[i % 3]) for i in range(n))


def exact_weight(k, n, group, gen):
    """A weight whose scales are powers of two, 2^-6 to 2^-3."""
    import torch
    W = Weight(k, n, group, gen)
    W.s = torch.exp2(torch.randint(-6, -2, W.s.shape, device="cuda", generator=gen).float()).half()
    W.v = W.w.double() * W.s.double().repeat_interleave(group, 0)[:k]
    return W


@pytest.mark.parametrize("rows", [1, 8, 9, 40, 64, 130])
@pytest.mark.parametrize("k,n,group", [(8192, 200, 128), (8191, 65, 32), (5001, 129, 64), (300, 1000, 32)])
def test_exact_sums(rows, k, n, group):
    """Small whole activations and scales that are powers of two: every sum,
    in any order, is a whole number of 2^-6 below 2^24 of them, so fp32 holds
    it exactly and the output is the exact sum rounded once, bit for bit. A
    lost or doubled row of K, or another group's scale, shows."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(k + rows)
    W = exact_weight(k, n, group, gen)
    packed = pack(k, n, group, W)
    x = make_x(rows, k, gen)
    x[:, :k] = torch.randint(-3, 4, (rows, k), device="cuda", generator=gen).half()
    x[:, k - 1] = 3.0  # the last row of K weighs in every output
    xd = x[:, :k].double()
    assert (xd.abs() @ W.v.abs()).max() * 64 < 2**24
    y = torch.empty(rows, n, device="cuda", dtype=torch.float16)
    T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y.data_ptr(), x_stride=x.stride(0))
    torch.cuda.synchronize()
    assert torch.equal(y, (xd @ W.v).half())


@pytest.mark.parametrize("rows", [1, 8, 40, 130])
@pytest.mark.parametrize("k,n,group", [(4096, 100, 128), (4095, 33, 32)])
def test_exact_gated_sums(rows, k, n, group):
    """The same of a gated pair: both sums are exact (17 bits), their product
    is rounded to fp32 and then to fp16, as here."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(k + rows + 1)
    A, B = exact_weight(k, n, group, gen), exact_weight(k, n, group, gen)
    packed = pack(k, n, group, A, B)
    x = make_x(rows, k, gen)
    x[:, :k] = torch.randint(-1, 2, (rows, k), device="cuda", generator=gen).half() / 16
    x[:, k - 1] = 0.0625
    xd = x[:, :k].double()
    assert max((xd.abs() @ M.v.abs()).max() for M in (A, B)) * 1024 < 2**24
    y = torch.empty(rows, n, device="cuda", dtype=torch.float16)
    T.linear_gated(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y.data_ptr(), activation=T.TL_ACT_RELU,
                   x_stride=x.stride(0))
    torch.cuda.synchronize()
    ref = torch.relu(xd @ A.v) * (xd @ B.v)
    assert torch.equal(y, ref.float().half())


@pytest.mark.parametrize("rows", [1, 8, 33, 64, 200])
@pytest.mark.parametrize("k,group", [(512, 32), (4096, 128), (8192, 64)])
@pytest.mark.parametrize("gated", [False, True])
def test_no_weight_is_rounded(rows, k, group, gated):
    """The outputs' rms error is the final rounding's alone. Next to that
    rounding (2.1e-4 of the value, rms) the fp32 sums add sqrt(k) 2^-23 at
    most (1.1e-5 at 8192: 0.2 %, in rms); weights rounded to fp16 first would
    add as much again (41 % in rms). The limit is 5 %."""
    import torch
    n = 20000 // rows + 7
    gen = torch.Generator(device="cuda").manual_seed(k + rows)
    A = Weight(k, n, group, gen)
    B = Weight(k, n, group, gen) if gated else None
    packed = pack(k, n, group, A, B)
    x = make_x(rows, k, gen)
    y = torch.empty(rows, n, device="cuda", dtype=torch.float16)
    xd = x[:, :k].double()
    ref = xd @ A.v
    if gated:
        T.linear_gated(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y.data_ptr(), activation=T.TL_ACT_NONE,
                       x_stride=x.stride(0))
        ref = ref * (xd @ B.v)
    else:
        T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y.data_ptr(), x_stride=x.stride(0))
    torch.cuda.synchronize()
    rms = (y.double() - ref).square().mean().sqrt()
    assert rms <= 1.05 * (ref.half().double() - ref).square().mean().sqrt()


@pytest.mark.parametrize("rows,k,n,group", [(3, 1 << 20, 65, 128), (33, 1 << 20, 40, 32), (2, 40, 1 << 22, 32),
                                            (40, 33, 1 << 22, 64), (1 << 20, 24, 9, 32)])
def test_the_largest_dimensions(rows, k, n, group):
    """k, n and rows at their documented limits, on sums that are exact."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(rows)
    W = Weight.__new__(Weight)
    W.w = torch.randint(-128, 128, (k, n), device="cuda", generator=gen, dtype=torch.int8)
    W.s = torch.full((-(-k // group), n), 0.125, device="cuda", dtype=torch.float16)
    W.s[:, ::2] = 0.25
    packed = pack(k, n, group, W)
    x = make_x(rows, k, gen)
    x[:, :k] = torch.randint(0, 50, (rows, k), device="cuda", generator=gen) == 0  # zeros and ones: |sum| < 2^21
    x[:, 0] = x[:, k - 1] = 1.0
    y = torch.full((rows + 1, n), 7.0, device="cuda", dtype=torch.float16)
    T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y.data_ptr(), x_stride=x.stride(0))
    torch.cuda.synchronize()
    scale = W.s[0].double()
    for j in range(0, n, 1 << 19):  # (the scales of a column are alike; its product is a whole number)
        part = x[:, :k].double() @ W.w[:, j:j + (1 << 19)].double() * scale[j:j + (1 << 19)]
        assert torch.equal(y[:rows, j:j + (1 << 19)], part.half())
    assert (y[rows] == 7.0).all()


@pytest.mark.parametrize("rows", [2, 33, 150])
def test_a_capture_that_forks_and_joins(rows):
    """A product captured behind two streams' kernels, one its input, one its
    residual, and read by kernels of both."""
    import torch
    k, n, group = 1024, 256, 64
    gen = torch.Generator(device="cuda").manual_seed(14)
    W = Weight(k, n, group, gen)
    packed = pack(k, n, group, W)
    x, x2 = make_x(rows, k, gen), make_x(rows, n, gen)
    P = Weight(n, n, group, gen)
    packed2 = pack(n, n, group, P)
    side = torch.cuda.Stream()

    def chain(out):
        main = torch.cuda.current_stream()
        res, y = out
        side.wait_stream(main)
        T.linear(x2.data_ptr(), rows, packed2.data_ptr(), n, n, group, res.data_ptr(), stream=side.cuda_stream)
        T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y[0].data_ptr(), stream=main.cuda_stream)
        main.wait_stream(side)
        T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y[1].data_ptr(), residual=res.data_ptr(),
                 stream=main.cuda_stream)
        side.wait_stream(main)
        T.linear(y[1].data_ptr(), rows, packed2.data_ptr(), n, n, group, y[2].data_ptr(), stream=side.cuda_stream)
        T.linear(y[1].data_ptr(), rows, packed2.data_ptr(), n, n, group, y[3].data_ptr(), residual=y[0].data_ptr(),
                 stream=main.cuda_stream)
        main.wait_stream(side)

    def fresh():
        return (torch.zeros(rows, n, device="cuda", dtype=torch.float16),
                torch.zeros(4, rows, n, device="cuda", dtype=torch.float16))

    ref, got = fresh(), fresh()
    chain(ref)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain(got)
    for _ in range(20):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    assert (ref[1].abs().amax((1, 2)) > 0).all()


def test_beside_prefill_attention():
    """Products of every row tile on two streams while a third runs the
    prefill kernel, which takes all of an SM's TMEM: each gives what it gives
    alone."""
    import torch
    from gpu_helpers import Run
    r = Run.create(1, 8, 2, 128, 16, 1024, 2)
    sid = r.allocate(1024)
    r.prefill(sid, 900, 5)
    gen = torch.Generator(device="cuda").manual_seed(15)
    q = torch.randn(900, 8, 128, device="cuda", generator=gen).half()
    o = torch.empty(12, 900, 8, 128, device="cuda", dtype=torch.float16)
    k, n, group = 2048, 1500, 128
    W = Weight(k, n, group, gen)
    packed = pack(k, n, group, W)
    jobs = []
    for rows in (4, 20, 32, 50, 64, 100, 300):
        x = make_x(rows, k, gen)
        ref = torch.empty(rows, n, device="cuda", dtype=torch.float16)
        T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, ref.data_ptr())
        jobs.append((rows, x, ref, torch.empty(12, rows, n, device="cuda", dtype=torch.float16)))
    alone = torch.empty_like(o[0])
    r.cache.prefill_attention(0, q.data_ptr(), alone.data_ptr(), [sid], [900])
    torch.cuda.synchronize()
    a, b, c = (torch.cuda.Stream() for _ in range(3))
    for i in range(12):
        r.cache.prefill_attention(0, q.data_ptr(), o[i].data_ptr(), [sid], [900], stream=a.cuda_stream)
        for j, (rows, x, _, y) in enumerate(jobs):
            T.linear(x.data_ptr(), rows, packed.data_ptr(), k, n, group, y[i].data_ptr(),
                     stream=(b if (i + j) % 2 else c).cuda_stream)
    torch.cuda.synchronize()
    r.cache.sync_check()
    assert all(torch.equal(o[i], alone) for i in range(12))
    for _, _, ref, y in jobs:
        assert all(torch.equal(y[i], ref) for i in range(12))
