"""Refusals of the W8A16 projections and of tl_token_logprobs, and the packed
sizes: what is decided on the host, before any device is looked at."""
import pytest

import tiny_llm_b200 as T

A = 0x10000  # a pointer that is never read: every call here is refused first


def status(call):
    with pytest.raises(T.TLError) as e:
        call()
    return type(e.value), str(e.value)


def test_packed_bytes():
    # tiles of 64 columns x blocks of 128 rows, each 8 KB and its scales
    assert T.linear_packed_bytes(128, 64, 128) == 8192 + 128
    assert T.linear_packed_bytes(129, 65, 64) == 4 * (8192 + 256)
    assert T.linear_packed_bytes(1, 1, 32) == 8192 + 512
    assert T.linear_packed_bytes(4096, 14336, 128, True) == 448 * 32 * 8320
    assert T.linear_packed_bytes(4096, 33, 128, True) == 2 * 32 * 8320  # 5 eights of each


@pytest.mark.parametrize("k,n,group", [(0, 8, 32), (8, 0, 32), (-1, 8, 32), (8, 8, 16), (8, 8, 0), (8, 8, 256),
                                       (1 << 21, 8, 32), (8, 1 << 23, 32)])
def test_shapes_refused(k, n, group):
    want = T.InvalidArgument if k <= 0 or n <= 0 else T.Unsupported
    assert status(lambda: T.linear_packed_bytes(k, n, group))[0] is T.Unsupported
    assert status(lambda: T.pack_linear_weight(A, A, k, n, group, A))[0] is want
    assert status(lambda: T.linear(A, 1, A, k, n, group, A))[0] is want
    assert status(lambda: T.linear_gated(A, 1, A, k, n, group, A))[0] is want


def test_pack_refusals():
    big = 1 << 40
    for args in [(0, A, big), (A, 0, big), (A, A, 0)]:
        assert "null" in status(lambda: T.pack_linear_weight(args[0], args[1], 64, 64, 32, args[2]))[1]
    assert "both" in status(lambda: T.pack_linear_weight(A, A, 64, 64, 32, big, w_up_ptr=A))[1]
    assert "both" in status(lambda: T.pack_linear_weight(A, A, 64, 64, 32, big, scales_up_ptr=A))[1]
    assert "aligned" in status(lambda: T.pack_linear_weight(A, A, 64, 64, 32, big + 8))[1]
    assert "aligned" in status(lambda: T.pack_linear_weight(A, A + 1, 64, 64, 32, big))[1]
    assert "overlap" in status(lambda: T.pack_linear_weight(A, big, 64, 64, 32, A + 1024))[1]
    assert "overlap" in status(lambda: T.pack_linear_weight(big, A, 64, 64, 32, A))[1]


@pytest.mark.parametrize("gated", [False, True])
def test_linear_refusals(gated):
    def call(x=A, rows=4, packed=A, k=64, n=64, group=32, y=A, **kw):
        (T.linear_gated if gated else T.linear)(x, rows, packed, k, n, group, y, **kw)

    assert "rows" in status(lambda: call(rows=-1))[1]
    assert status(lambda: call(rows=(1 << 20) + 1))[0] is T.Unsupported
    call(rows=0)  # nothing to do
    call(x=0, y=0, packed=0, rows=0)
    assert "input is null" in status(lambda: call(x=0))[1]
    assert "output is null" in status(lambda: call(y=0))[1]
    assert "packed weights are null" in status(lambda: call(packed=0))[1]
    assert "aligned" in status(lambda: call(x=A + 8))[1]
    assert "aligned" in status(lambda: call(packed=A + 4))[1]
    assert "aligned" in status(lambda: call(y=A + 1))[1]
    assert "aligned" in status(lambda: call(bias=A + 1))[1]
    assert "x_stride" in status(lambda: call(x_stride=56))[1]
    assert "x_stride" in status(lambda: call(x_stride=68))[1]
    assert "x_stride" in status(lambda: call(k=63))[1]  # rows of 63 are not 16-byte aligned
    assert "strides" in status(lambda: call(y_stride=63))[1]
    assert "activation" in status(lambda: call(activation=5))[1]
    assert "activation" in status(lambda: call(activation=-1))[1]
    if not gated:
        assert "strides" in status(lambda: call(residual=A, residual_stride=60))[1]


def test_residual_in_place_keeps_the_stride():
    """Row r of the residual would be another row's output otherwise."""
    def call(rows, **kw):
        T.linear(A, rows, A, 64, 64, 32, A, residual=A, **kw)

    assert "in place" in status(lambda: call(4, residual_stride=72))[1]
    assert "in place" in status(lambda: call(9, y_stride=128))[1]
    call(0, residual_stride=72)  # nothing to do


def test_logprob_refusals():
    def call(logits=A, rows=4, vocab=100, tokens=A, lp=A, **kw):
        T.token_logprobs(logits, rows, vocab, tokens, lp, **kw)

    assert "rows" in status(lambda: call(rows=-1))[1]
    assert "vocab" in status(lambda: call(vocab=0))[1]
    assert status(lambda: call(dtype=3))[0] is T.Unsupported
    assert status(lambda: call(top_n=65))[0] is T.Unsupported
    assert status(lambda: call(top_n=-1))[0] is T.Unsupported
    call(rows=0)
    assert "logits is null" in status(lambda: call(logits=0))[1]
    assert "tokens is null" in status(lambda: call(tokens=0))[1]
    assert "every output" in status(lambda: call(lp=0))[1]
    assert "every output" in status(lambda: call(lp=0, top_n=3))[1]
    assert "every output" in status(lambda: call(lp=0, top_n=0, top_tokens_ptr=A))[1]
    assert "row_stride" in status(lambda: call(row_stride=99))[1]
    assert "row_stride" in status(lambda: call(row_stride=-100))[1]
    assert "aligned" in status(lambda: call(logits=A + 1))[1]
    assert "aligned" in status(lambda: call(logits=A + 2, dtype=T.TL_F32))[1]
    assert "aligned" in status(lambda: call(tokens=A + 2))[1]


def test_logprob_rows_whose_indices_would_wrap():
    """The search through a slice steps by 512 elements: past 2^31 from here on."""
    for vocab in (2**31 - 1023, 2**31 - 1):
        kind, text = status(lambda: T.token_logprobs(A, 1, vocab, A, A))
        assert kind is T.Unsupported and "vocab" in text


def test_without_a_device():
    """Where there is no device the calls say so."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("a device is present")
    assert status(lambda: T.linear(A, 1, A, 64, 64, 32, A))[0] is T.NoDevice
    assert status(lambda: T.pack_linear_weight(1 << 40, 1 << 41, 64, 64, 32, A))[0] is T.NoDevice
    assert status(lambda: T.token_logprobs(A, 1, 100, A, A))[0] is T.NoDevice
