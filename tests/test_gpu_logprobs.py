"""tl_token_logprobs on the device against log_softmax in float64.

Tolerance. With z = (x - max) / T and l = sum exp z: z and its scale carry
two fp32 roundings (2^-24 of |z| each, and one more of the product), 2^z the
hardware's two units, a thread's running sums one unit an addition and one a
rescaling; a row's weights are positive, so log l is off by at most the
relative error of l, below (128 + 30) 2^-23 for rows of up to 160000 elements
over 512 threads and more (at most 320 additions a thread in half-precision
types, taken at random signs) plus |z| 2^-22 of the terms that count. Taken
together: 4e-6 + 4e-7 |z| for log probabilities, ten times the first for the
entropy, whose terms weigh |z|."""
import numpy as np
import pytest

import conftest
import tiny_llm_b200 as T

pytestmark = pytest.mark.gpu

DT = {"f16": T.TL_F16, "bf16": T.TL_BF16, "f32": T.TL_F32}


@pytest.fixture(autouse=True)
def _need_gpu():
    if not conftest.cuda_available():
        pytest.skip("no CUDA device")


def torch_type(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def call(logits, tokens, top, dtype, temperature=1.0, stride=None, rows=None, vocab=None):
    """(logprobs, entropy, top tokens, top logprobs), guarded on both sides."""
    import torch
    rows, vocab = rows or logits.shape[0], vocab or logits.shape[1]
    lp, ent = (torch.full((rows + 2,), 99.0, device="cuda") for _ in range(2))
    tt = torch.full((rows * top + 2,), 99, device="cuda", dtype=torch.int32)
    tl = torch.full((rows * top + 2,), 99.0, device="cuda")
    T.token_logprobs(logits.data_ptr(), rows, vocab, tokens.data_ptr(), lp[1:].data_ptr(), ent[1:].data_ptr(), top,
                     tt[1:].data_ptr(), tl[1:].data_ptr(), DT[dtype],
                     logits.stride(0) if stride is None else stride, temperature)
    torch.cuda.synchronize()
    for t in (lp, ent, tt, tl):
        assert t[0] == 99 and t[-1] == 99
    return lp[1:-1], ent[1:-1], tt[1:-1].view(rows, top), tl[1:-1].view(rows, top)


def check(logits, tokens, top, dtype, temperature=1.0, **kw):
    import torch
    lp, ent, tt, tl = call(logits, tokens, top, dtype, temperature, **kw)
    x = logits.double() / max(temperature, 1e-5)
    rows, vocab = x.shape
    # relative to the largest: next to a type's lowest value log l would be lost even in 64 bits
    z = x - x.max(1, keepdim=True).values
    lsm = z - torch.logsumexp(z, 1, keepdim=True)
    z = torch.where(z > float("-inf"), z, 0.0)
    t = tokens.long()
    want = torch.where(t < 0, 0.0, lsm.gather(1, t.clamp(0, vocab - 1)[:, None])[:, 0])
    tol = 4e-6 + 4e-7 * z.gather(1, t.clamp(0, vocab - 1)[:, None])[:, 0].abs()
    same = (lp.double() == want) | ((lp.double() - want).abs() <= tol)
    assert same.all(), f"{lp[~same][:4]} {want[~same][:4]}"
    p = lsm.exp()
    want_ent = -torch.where(p > 0, p * lsm, 0.0).sum(1)
    assert ((ent.double() - want_ent).abs() <= 4e-5).all(), f"{(ent.double() - want_ent).abs().max()}"
    # the stable descending order's first ones, as far as they are allowed
    order = torch.sort(logits.float() + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    ok = logits.gather(1, order) > float("-inf")
    order = torch.where(ok, order, -1).to(torch.int32)
    if order.shape[1] < top:
        order = torch.nn.functional.pad(order, (0, top - order.shape[1]), value=-1)
    assert torch.equal(tt, order)
    vals = torch.where(order >= 0, lsm.gather(1, order.long().clamp(min=0)), float("-inf"))
    zt = torch.where(order >= 0, z.gather(1, order.long().clamp(min=0)), 0.0)
    assert ((tl.double() == vals) | ((tl.double() - vals).abs() <= 4e-6 + 4e-7 * zt.abs())).all()


def make(rows, vocab, dtype, seed, pad=0, spread=3.0):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.full((rows, vocab + pad), float("inf"), device="cuda", dtype=torch_type(dtype))  # never read
    buf[:, :vocab] = (torch.randn(rows, vocab, device="cuda", generator=gen) * spread).to(torch_type(dtype))
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=gen).to(torch.int32)
    return buf[:, :vocab], tokens


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,pad", [(1, 1, 0), (3, 2, 1), (2, 7, 3), (1, 8, 0), (5, 31, 2), (4, 1000, 5),
                                            (1, 4097, 0), (9, 32000, 8), (1, 128256, 0), (2, 151937, 1), (300, 513, 3),
                                            (40, 50257, 1)])
def test_sizes(dtype, rows, vocab, pad):
    check(*make(rows, vocab, dtype, rows + vocab, pad), top=min(8, 64), dtype=dtype)


@pytest.mark.parametrize("top", [0, 1, 2, 20, 63, 64])
@pytest.mark.parametrize("rows,vocab", [(1, 128256), (3, 50), (160, 9000)])
def test_alternatives(top, rows, vocab):
    check(*make(rows, vocab, "f16", top), top=top, dtype="f16")


@pytest.mark.parametrize("temperature", [0.0, 0.05, 0.7, 1.0, 3.0])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_temperature(temperature, dtype):
    import torch
    logits, tokens = make(4, 20000, dtype, 11)
    if temperature == 0.0:  # clamped to 1e-5: everything on the largest
        logits[:, 77] = 40.0
        lp, ent, tt, tl = call(logits, torch.full_like(tokens, 77), 2, dtype, 0.0)
        assert (lp == 0).all() and (ent == 0).all() and (tt[:, 0] == 77).all() and (tl[:, 0] == 0).all()
    elif temperature == 0.05:
        # |z| reaches 500: probabilities below 2^-149 are 0 and the log
        # probabilities of the tail keep 4e-7 |z|
        check(logits, tokens, 5, dtype, temperature)
    else:
        check(logits, tokens, 5, dtype, temperature)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [40, 30000, 128256])
def test_ties(dtype, vocab):
    """Equal logits are listed by index: few values, all equal, +0 and -0."""
    import torch
    logits, tokens = make(4, vocab, dtype, 3)
    logits[0] = (logits[0].float() / 2).round().to(logits.dtype)  # a handful of values
    logits[1] = 1.5
    logits[2] = torch.where(torch.arange(vocab, device="cuda") % 3 == 1, 0.0, -0.0).to(logits.dtype)
    logits[3] = -7.0
    logits[3, vocab // 2:] = -6.5
    check(logits, tokens, 33, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [9, 5000, 128256])
def test_masks(dtype, vocab):
    """-inf, the type's lowest value, rows with few allowed tokens and none."""
    import torch
    logits, tokens = make(8, vocab, dtype, 4)
    low = torch.finfo(logits.dtype).min
    logits[0, 1:] = float("-inf")      # one allowed
    tokens[0] = 0
    logits[1, : vocab - 2] = float("-inf")
    tokens[1] = 0                      # a masked one is asked for
    logits[2, ::2] = low
    logits[3] = low                    # nothing but the lowest: uniform
    logits[4] = low
    logits[4, 3] = float("-inf")
    tokens[4] = 3
    logits[5, ::2] = float("-inf")
    logits[5, 1::2] = low              # lowest and -inf
    logits[6, : vocab // 2] = float("-inf")
    tokens[7] = -5                     # padding
    check(logits, tokens, 6, dtype)
    none = torch.full((3, vocab), float("-inf"), device="cuda", dtype=logits.dtype)
    lp, ent, tt, tl = call(none, torch.tensor([0, -1, vocab], device="cuda", dtype=torch.int32), 4, dtype)
    assert lp[0] == float("-inf") and lp[1] == 0 and lp[2].isnan()
    assert (ent == 0).all() and (tt == -1).all() and (tl == float("-inf")).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [11, 128256])
def test_nan_and_inf_rows(dtype, vocab):
    import torch
    logits, tokens = make(5, vocab, dtype, 5)
    logits[0, vocab - 1] = float("nan")
    logits[1, 0] = float("inf")
    logits[2] = float("nan")
    logits[3, 2] = float("nan")
    tokens[3] = -1
    lp, ent, tt, tl = call(logits, tokens, 3, dtype)
    assert lp[:3].isnan().all() and lp[3] == 0 and ent[:4].isnan().all()
    assert (tt[:4] == -1).all() and tl[:4].isnan().all()
    check(logits[4:], tokens[4:], 3, dtype)  # the row beside them is itself


def test_extreme_values():
    """fp32 logits near the type's ends, differences that overflow."""
    import torch
    big = torch.finfo(torch.float32).max
    logits = torch.full((3, 1000), -big, device="cuda")
    logits[0, 5] = big
    logits[1, 5] = 1e30
    logits[1, 7] = 1e30
    logits[2, :] = big
    lp, ent, tt, tl = call(logits, torch.tensor([5, 7, 999], device="cuda", dtype=torch.int32), 2, "f32")
    ref = torch.tensor([0.0, -np.log(2.0), -np.log(1000.0)])
    assert ((lp.cpu() - ref).abs() < 4e-6).all() and ((ent.cpu() + ref).abs() < 4e-5).all()
    assert tt.tolist() == [[5, 0], [5, 7], [0, 1]]


def test_shared_row_and_given_outputs():
    """row_stride 0 shares one row; outputs that are not wanted are null."""
    import torch
    logits, _ = make(1, 3001, "f16", 6)
    tokens = torch.arange(10, device="cuda", dtype=torch.int32)
    lp, ent, tt, tl = call(logits, tokens, 2, "f16", stride=0, rows=10, vocab=3001)
    one = torch.log_softmax(logits.double(), 1)[0]
    assert ((lp.double() - one[:10]).abs() < 1e-5).all() and (ent == ent[0]).all() and (tt == tt[0]).all()
    out = torch.zeros(10, device="cuda")
    T.token_logprobs(logits.data_ptr(), 10, 3001, tokens.data_ptr(), out.data_ptr(), row_stride=0)
    e2 = torch.zeros(10, device="cuda")
    T.token_logprobs(logits.data_ptr(), 10, 3001, 0, 0, e2.data_ptr(), row_stride=0)
    t2 = torch.zeros(10, 2, device="cuda", dtype=torch.int32)
    T.token_logprobs(logits.data_ptr(), 10, 3001, 0, 0, 0, 2, t2.data_ptr(), 0, row_stride=0)
    torch.cuda.synchronize()
    assert torch.equal(out, lp) and torch.equal(e2, ent) and torch.equal(t2, tt)


def test_far_rows():
    """Row offsets past 2^31 elements."""
    import torch
    vocab, stride = 1000, 1 << 28
    buf = torch.empty(9 * stride + vocab, device="cuda", dtype=torch.float16)
    rows = torch.as_strided(buf, (10, vocab), (stride, 1))
    rows.copy_(torch.randn(10, vocab, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)))
    tokens = torch.arange(10, device="cuda", dtype=torch.int32)
    lp, _, tt, _ = call(rows, tokens, 1, "f16")
    ref = torch.log_softmax(rows.double(), 1)
    assert ((lp.double() - ref[torch.arange(10), torch.arange(10)]).abs() < 1e-5).all()
    assert torch.equal(tt[:, 0].long(), rows.argmax(1))


def test_same_results_every_run_and_in_a_graph():
    import torch
    logits, tokens = make(6, 128256, "f16", 9)
    first = call(logits, tokens, 20, "f16")
    lp, ent = torch.zeros(6, device="cuda"), torch.zeros(6, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        T.token_logprobs(logits.data_ptr(), 6, 128256, tokens.data_ptr(), lp.data_ptr(), ent.data_ptr(),
                         stream=torch.cuda.current_stream().cuda_stream)
    graph.replay()
    again = call(logits, tokens, 20, "f16")
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    assert torch.equal(lp, first[0]) and torch.equal(ent, first[1])


@pytest.mark.parametrize("dtype,temperature", [("f16", 1e5), ("bf16", 3e37), ("f32", 3e37)])
@pytest.mark.parametrize("vocab", [9, 5000])
def test_masks_at_a_temperature_where_the_lowest_value_weighs(dtype, temperature, vocab):
    """The type's lowest value then has a probability of its own; -inf never.

    At 5000 tokens (10 elements a thread, 9 levels of joins, logarithms up to
    12.3 in base 2) the roundings add up to 3.1e-6, below check()'s 4e-6."""
    import torch
    logits, tokens = make(5, vocab, dtype, 21)
    low, nothing = torch.finfo(logits.dtype).min, float("-inf")
    logits[0, ::2] = low
    logits[1, ::2] = nothing
    logits[2, ::3] = low
    logits[2, 1::3] = nothing
    logits[3] = low
    logits[3, 0] = nothing
    tokens[0], tokens[1], tokens[2], tokens[3] = 0, 0, 0, 1
    check(logits, tokens, 5, dtype, temperature)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [130, 300, 890, 1024])
@pytest.mark.parametrize("top", [2, 20, 64])
def test_many_candidates(dtype, vocab, top):
    """Short rows and ties, whose list of candidates is long: few values, one
    value, both zeros, masks that leave fewer than top."""
    import torch
    logits, tokens = make(7, vocab, dtype, 31)
    logits[1] = (logits[1].float() / 2).round().to(logits.dtype)
    logits[2] = 3.25
    logits[3] = torch.where(torch.arange(vocab, device="cuda") % 3 == 1, 0.0, -0.0).to(logits.dtype)
    logits[4, 1:] = float("-inf")
    logits[5] = torch.finfo(logits.dtype).min
    logits[5, vocab // 2:] = -1.0
    logits[6, : vocab - 3] = float("-inf")
    tokens[4], tokens[5] = 0, vocab - 1
    check(logits, tokens, top, dtype)


@pytest.mark.parametrize("rows,vocab,dtype,top", [(300, 150001, "f32", 20), (300, 150001, "f32", 2), (300, 300007, "f16", 9),
                                                  (300, 30000, "f16", 5), (300, 30000, "f32", 64)])
def test_long_slices_looked_at_again(rows, vocab, dtype, top):
    """Slices of one batch of loads a thread to more than the kept maxima; the
    largest sit together in one thread's elements of some rows."""
    import torch
    logits, tokens = make(rows, vocab, dtype, 41)
    n = 16 // logits.element_size()
    for r in range(0, rows, 7):  # the same thread's vectors, batch after batch
        at = torch.arange(n * 3, vocab - 1, n * 256 * 8, device="cuda")[:top]
        logits[r, at] = 30.0 - torch.arange(at.numel(), device="cuda").to(logits.dtype)
    check(logits, tokens, top, dtype)


@pytest.mark.parametrize("temperature", [0.0, 2e-5, 4e-5])
@pytest.mark.parametrize("rows,vocab", [(1, 700), (1, 128256), (300, 1024), (300, 40003)])
def test_fp16_large_logits_at_the_lowest_temperatures(rows, vocab, temperature):
    """m log2(e) / T passes 2^31 (0 is clamped to 1e-5), where its fp32 rounding
    is hundreds: maxima of both signs to the type's ends, ties at the maximum,
    threads whose own maximum lies anywhere below it."""
    import torch
    maxima = [15104.0, 20000.0, 40000.0, 65504.0, -15104.0, -40000.0, -65472.0, 30000.0]
    gen = torch.Generator(device="cuda").manual_seed(51)
    for first in range(len(maxima) if rows == 1 else 1):
        top = torch.tensor([maxima[(first + r) % len(maxima)] for r in range(rows)], device="cuda")[:, None]
        body = -65504.0 + torch.rand(rows, vocab, device="cuda", generator=gen) * (top + 65504.0)
        near = torch.randn(rows, vocab, device="cuda", generator=gen) * 3.0
        narrow = (torch.arange(rows, device="cuda")[:, None] % 3 == 1) & (top > 0)
        logits = torch.minimum(torch.where(narrow, near, body), top).half()
        logits[:, 5:vocab:331] = top.half()  # ties
        tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=gen).to(torch.int32)
        tokens[::2] = 5
        check(logits, tokens, 8, "f16", temperature)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("temperature", [2.0, 4.0, 3e37, 1e38, 3e38])
def test_differences_past_the_types_end(dtype, temperature):
    """Logits whose difference overflows fp32 although, divided by T, it does
    not: the small one then has a log probability, at T near 1e38 a weight too.
    (Above 8e37 1 / T is subnormal: half a unit of it is 2.2e-7 of the value at
    3e38, of |z| up to 3.3 in base 2 7e-7, inside check()'s 4e-6 + 4e-7 |z|.)"""
    import torch
    logits, _ = make(6, 700, dtype, 61)
    big = torch.finfo(logits.dtype).max
    logits[0] = -big
    logits[0, 5] = big
    logits[1, ::2], logits[1, 1::2] = big, -big
    logits[2, ::3], logits[2, 1::3] = big * 0.75, -big * 0.625
    logits[3, 9] = big
    logits[4] = -big
    logits[4, 600:] = big
    logits[5, 3], logits[5, 4], logits[5, 5] = big, -big, float("-inf")
    tokens = torch.tensor([0, 1, 1, 4, 10, 4], device="cuda", dtype=torch.int32)
    check(logits, tokens, 4, dtype, temperature)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [9, 5000])
def test_infinite_temperature_is_uniform(dtype, vocab):
    """softmax(logits / inf): the same for every finite logit, none for -inf."""
    import torch
    logits, _ = make(3, vocab, dtype, 62)
    big = torch.finfo(logits.dtype).max
    logits[0, 1], logits[0, 2] = big, -big
    logits[1, ::2] = float("-inf")
    logits[2] = float("-inf")
    tokens = torch.tensor([2, 1, 0], device="cuda", dtype=torch.int32)
    lp, ent, tt, tl = call(logits, tokens, 3, dtype, float("inf"))
    allowed = torch.tensor([vocab, vocab // 2], dtype=torch.float64)
    assert ((lp[:2].double().cpu() + allowed.log()).abs() <= 4e-6).all()
    assert ((ent[:2].double().cpu() - allowed.log()).abs() <= 4e-5).all()
    assert ((tl[:2].double().cpu() + allowed.log()[:, None]).abs() <= 4e-6).all()
    assert lp[2] == float("-inf") and ent[2] == 0 and (tt[2] == -1).all()


def test_the_longest_row():
    """As many equal logits as a row may have: the list of candidates
    overflows, and the search in its place steps past the last index. (The
    sums are whole numbers; the logarithm's and the product's roundings are
    2.3e-6 at 21.5.)"""
    import torch
    vocab = 2**31 - 1024
    logits = torch.full((1, vocab), 1.0, device="cuda", dtype=torch.float16)
    tokens = torch.tensor([vocab - 1], device="cuda", dtype=torch.int32)
    lp, ent, tt, tl = call(logits, tokens, 2, "f16")
    want = -np.log(vocab)
    assert abs(lp.item() - want) <= 4e-6 and abs(ent.item() + want) <= 4e-5
    assert tt.tolist() == [[0, 1]] and (tl.double() - want).abs().max() <= 4e-6


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_many_short_rows(dtype):
    """2^20 rows of a few logits."""
    import torch
    rows, vocab = 1 << 20, 5
    logits, tokens = make(rows, vocab, dtype, 71, pad=2)
    lp, ent, tt, tl = call(logits, tokens, 2, dtype)
    lsm = torch.log_softmax(logits.double(), 1)
    assert ((lp.double() - lsm.gather(1, tokens.long()[:, None])[:, 0]).abs() <= 1e-5).all()
    assert ((ent.double() + (lsm.exp() * lsm).sum(1)).abs() <= 4e-5).all()
    order = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :2]
    assert torch.equal(tt.long(), order)
    assert ((tl.double() - lsm.gather(1, order)).abs() <= 1e-5).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("temperature", [2e36, 1e38])
@pytest.mark.parametrize("rows,vocab", [(2, 128256), (300, 20011)])
def test_long_rows_of_the_types_ends(dtype, temperature, rows, vocab):
    """Differences past fp32's range over many batches, split rows and joins."""
    import torch
    logits, tokens = make(rows, vocab, dtype, 63)
    big = torch.finfo(logits.dtype).max
    gen = torch.Generator(device="cuda").manual_seed(64)
    u = torch.rand(rows, vocab, device="cuda", generator=gen) * 2 - 1
    logits[:] = (u * big).to(logits.dtype)
    logits[:, 7::5] = float("-inf")
    logits[:, 11], logits[:, vocab - 3] = big, -big
    tokens[::2] = vocab - 3
    check(logits, tokens, 8, dtype, temperature)


@pytest.mark.parametrize("dtype,temperature", [("bf16", 1.0), ("f32", 1.0), ("f16", 1e4)])
@pytest.mark.parametrize("rows,vocab", [(300, 128256), (450, 160001)])
def test_rows_of_alike_weights(dtype, temperature, rows, vocab):
    """The largest logit in every thread's first vector and one value for all
    the others, 500 to 625 to a thread, so that every addition to a running sum
    could round the same way: 7.7e-6 of it, one by one. By batches of at most 64 it is 1e-6, and with 16
    batches, 11 joins (2^-24 each, 1.6e-6) and the logarithm's roundings (at 12:
    1.2e-6) 3.8e-6, below check()'s 4e-6 + 4e-7 |z|."""
    import torch
    logits, tokens = make(rows, vocab, dtype, 81)
    level = -(torch.arange(rows, device="cuda") % 50 + 14).float() / 64  # weights 0.37 to 0.8
    logits[:] = (level * temperature)[:, None].to(logits.dtype)
    logits[:, :2048] = 0.0
    check(logits, tokens, 0, dtype, temperature)
