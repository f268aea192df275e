"""A step that its buffers were not made for is refused before anything is launched (no GPU is needed to be refused)."""
import pytest
import torch

from rocwmma_amd import decode_step as D


def _layer():
    layer = object.__new__(D.AttentionLayer)  # sizes only: neither weights nor a cache
    layer.hidden, layer.torch_type = 64, torch.float16
    layer.total_tokens, layer.batch, layer.max_tokens, layer.max_kv = 6, 2, 4, 100
    return layer


def _step(**change):
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)
    step = dict(x=torch.zeros(6, 64, dtype=torch.float16), positions=i32(6), slots=i32(6), table=torch.zeros(2, 7, dtype=torch.int32), q_start=i32(3), kv_len=i32(2),
                mask=torch.zeros(6, 1, dtype=torch.int64))
    step.update(change)
    return step


def test_a_step_of_the_reserved_size_is_taken():
    layer = _layer()
    layer._holds(**_step())
    layer._holds(**_step(mask=None, q_start=torch.zeros(9, dtype=torch.int32), kv_len=torch.zeros(9, dtype=torch.int32)))
    one = torch.zeros(1, dtype=torch.int32)
    layer._holds(**_step(x=torch.zeros(1, 64, dtype=torch.float16), positions=one, slots=one, table=torch.zeros(1, 7, dtype=torch.int32)))


@pytest.mark.parametrize("change", [
    dict(x=torch.zeros(7, 64, dtype=torch.float16), positions=torch.zeros(7, dtype=torch.int32), slots=torch.zeros(7, dtype=torch.int32), mask=None),  # more than reserved
    dict(table=torch.zeros(3, 7, dtype=torch.int32), q_start=torch.zeros(4, dtype=torch.int32), kv_len=torch.zeros(3, dtype=torch.int32)),
    dict(positions=torch.zeros(5, dtype=torch.int32)), dict(positions=torch.zeros(7, dtype=torch.int32)), dict(slots=torch.zeros(5, dtype=torch.int32)),
    dict(q_start=torch.zeros(2, dtype=torch.int32)), dict(kv_len=torch.zeros(1, dtype=torch.int32)),
    dict(mask=torch.zeros(5, 1, dtype=torch.int64)), dict(mask=torch.zeros(6, dtype=torch.int64)),
    dict(x=torch.zeros(6, 72, dtype=torch.float16)), dict(x=torch.zeros(6, 128, dtype=torch.float16)[:, ::2]), dict(x=torch.zeros(6, 64, dtype=torch.bfloat16)),
    dict(x=torch.zeros(6, 72, dtype=torch.float16)[:, :64])])
def test_a_step_that_does_not_fit_is_refused(change):
    with pytest.raises(ValueError):
        _layer().step(**_step(**change))
