"""The binding's view of the layer operators' buffers, without a GPU: tensors that a call would read at the wrong
places are refused before any call."""
import numpy as np
import pytest

import turbo_decode_tail as T

torch = pytest.importorskip("torch")


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
