"""The binding's view of the layer operators' buffers, without a GPU: strides of heads that are slices of wider
rows, and tensors that a call would read at the wrong places, which are refused before any call."""
import numpy as np
import pytest

import turbo_decode_tail as T

torch = pytest.importorskip("torch")
F32, BF16 = T.TURBO_HIDDEN_F32, T.TURBO_HIDDEN_BF16


class Library:
    def __getattr__(self, name):
        return lambda *args: pytest.fail(f"{name} was called")


def cache():
    """A binding object without a handle: a refusal comes before the library is called."""
    c = object.__new__(T.KvCache)
    c.lib, c.h = Library(), None
    return c


def zeros(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_strides_of_slices():
    wide = zeros(6, 10, 64)
    assert T._stride(wide, F32) == 0 and T._stride(None, F32) == 0 and T._stride(12345, F32) == 0
    assert T._stride(wide[:, 2:6], F32) == 640
    assert T._stride(wide.bfloat16()[:, 2:6], BF16) == 640
    assert T._stride(wide[:, 3:4], F32) == 640
    assert T._stride(wide[::2], F32) == 1280                       # every other token
    assert T._stride(wide.view(6, 640)[:, 64:192], F32) == 640     # heads and values in one dimension
    assert T._stride(zeros(2, 3, 10, 64)[:, :, 1:5], F32) == 640   # [batch][q_len][heads][head_dim]
    assert T._stride(zeros(1, 10, 64)[:, 1:5], F32) == 0           # one token: any stride
    assert T._stride(zeros(2, 1, 10, 64)[:, :, 1:5], F32) == 640
    assert T._stride(zeros(4, 1, 64).transpose(0, 1).contiguous().transpose(0, 1), F32) == 0


@pytest.mark.parametrize("t,word", [
    (zeros(6, 10, 64).transpose(0, 1), "contiguous"),              # heads outside tokens
    (zeros(6, 10, 128)[:, :, :64], "contiguous"),                  # a gap between heads
    (zeros(6, 10, 128)[:, :, ::2], "contiguous"),
    (zeros(6, 1280)[:, ::2], "contiguous"),
    (zeros(1280)[::2], "contiguous"),
    (zeros(1, 4, 64).expand(6, 4, 64), "overlap"),                 # one token for all
    (zeros(640).as_strided((6, 2, 64), (64, 64, 1)), "overlap"),
    (zeros(4, 3, 10, 64)[:, :2], "one stride"),                    # two of three queries of each sequence
    (zeros(3, 2, 10, 64).transpose(0, 1), "one stride"),
])
def test_refused_layouts(t, word):
    with pytest.raises(ValueError, match=word):
        T._stride(t, F32)


def test_another_element_size_is_refused():
    x, sl = zeros(4, 2, 64, dtype=torch.bfloat16), zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="element size"):
        cache().write(x, x, sl, 4)  # dtype is FP32 unless given: the call would read past the end
    with pytest.raises(ValueError, match="element size"):
        cache().read(sl, 4, zeros(4, 2, 64), None, dtype=BF16)
    with pytest.raises(ValueError, match="element size"):
        T.Rotary.make_inputs(4, q=x, q_heads=2, positions=sl, q_out=x)
    with pytest.raises(ValueError, match="element size"):
        T.KvCache.make_attention_inputs(4, q=x, out=x, q_heads=2, kv_len=sl, max_kv_len=1, scale=1.0)


def attention(**kw):
    q = zeros(2, 4, 64)
    a = dict(q=q, out=torch.empty_like(q), q_heads=4, kv_len=zeros(2, dtype=torch.int32), max_kv_len=9, scale=1.0,
             pages=zeros(2, 4, dtype=torch.int32), prefix_len=5, prefix_pages=zeros(1, dtype=torch.int32))
    a.update(kw)
    return T.KvCache.make_attention_inputs(2, **a)


def test_a_slice_of_a_wider_page_table_is_refused():
    table = torch.arange(24, dtype=torch.int32).view(2, 12)
    with pytest.raises(ValueError, match="contiguous 32-bit"):
        attention(pages=table[:, :4])
    assert attention(pages=table[:, :4].contiguous()).page_stride == 4
    assert attention(pages=table).page_stride == 12


@pytest.mark.parametrize("bad", [zeros(2, dtype=torch.int64), zeros(2), zeros(4, dtype=torch.int32)[::2]])
def test_ids_of_another_kind_are_refused(bad):
    x = zeros(2, 2, 64)
    for call in (lambda: attention(kv_len=bad), lambda: attention(prefix_pages=bad), lambda: attention(pages=bad[None]), lambda: cache().write(x, x, bad, 2),
                 lambda: cache().read(bad, 2, x, None), lambda: T.Rotary.make_inputs(2, q=x, q_heads=2, positions=bad, q_out=x),
                 lambda: T.Rotary.make_inputs(2, k=x, v=x, kv_heads=2, slots=bad)):
        with pytest.raises(ValueError, match="32-bit integers"):
            call()


@pytest.mark.parametrize("w", [np.ones(64, np.float32), np.ones(128, np.uint16)[::2]])
def test_norm_weights_of_another_kind_are_refused(w):
    with pytest.raises(ValueError, match="BF16"):
        T.Rotary(64, q_norm=w)
