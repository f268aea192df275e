"""Arrays of positions, slots, pages and lengths that a kernel would read as what they are not are refused by the Python calls.  (Host tensors that pass for device memory: nothing
is launched.)"""
import numpy as np
import pytest
import torch

import rocwmma_amd as R


class _Library:
    """what the calls reach instead of the library: it keeps what it was given"""

    def __init__(self):
        self.args = []

    def r355_rope(self, args, stream):
        self.args.append(R._ROPE_ARGS.unpack(args))
        return 0

    def r355_tree_attention(self, args, stream):
        self.args.append(args._obj)
        return 0

    def r355_w4_matmul(self, args, stream):
        self.args.append(args._obj)
        return 0


class _OnDevice(torch.Tensor):
    is_cuda = True


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32).as_subclass(_OnDevice)


def _i64(*shape):
    return torch.zeros(*shape, dtype=torch.int64).as_subclass(_OnDevice)


@pytest.fixture
def library(monkeypatch):
    library = _Library()
    monkeypatch.setattr(R, "lib", lambda: library)
    return library


def _rope(**change):
    a = dict(positions=_i32(4), turns=_i64(32), slots=_i32(4), slot_count=9)
    a.update(change)
    R.rope(R.F16, R.ROPE_HALF, 4, 64, 64, [R.rope_part(0x1000, 0x2000, 2, (128, 64), (128, 64), to_slots=True)], **a)


def _tree(**change):
    a = dict(table=_i32(3, 7), q_start=_i32(4), kv_len=_i32(3), mask=_i64(6, 2), mask_words=2, max_kv=7 * 16)
    a.update(change)
    R.tree_attention(R.F16, 3, 6, 4, 2, 64, 0x1000, 0x2000, 0x3000, 0x4000, page_size=16, pages=30, max_tokens=2, **a)


def _pinned(t):
    """a host tensor that says it is pinned"""
    t = t.as_subclass(type("Pinned", (torch.Tensor,), {"is_pinned": lambda self: True}))
    assert not t.is_cuda
    return t


def test_arrays_of_the_right_kind_are_taken(library):
    p, t = _i32(9), _i64(32)
    _rope(positions=p, turns=t)
    _rope(positions=p[3:7], turns=t.numpy().ctypes.data, slots=None)
    _rope(positions=_pinned(torch.zeros(4, dtype=torch.int32)))
    assert [(a[36], a[37]) for a in library.args[:2]] == [(p.data_ptr(), t.data_ptr()), (p.data_ptr() + 12, t.data_ptr())]
    _tree()
    _tree(mask=None, mask_words=0, q_start=0x5000, kv_len=_i32(12))
    _tree(table=0x6000, table_stride=7)
    _tree(table=_i32(21), table_stride=7)


@pytest.mark.parametrize("change", [dict(positions=_i64(4)), dict(slots=_i64(4)), dict(turns=_i32(64)), dict(positions=_i32(3)), dict(slots=_i32(3)), dict(turns=_i64(31)),
                                    dict(positions=_i32(8)[::2]), dict(positions=torch.zeros(4).as_subclass(_OnDevice)), dict(positions=torch.zeros(4, dtype=torch.int32)),
                                    dict(slots=np.zeros(4, np.int32)), dict(turns=np.zeros(32, np.uint64))])
def test_rope_refuses(library, change):
    with pytest.raises(ValueError):
        _rope(**change)
    assert not library.args


@pytest.mark.parametrize("change", [dict(table=_i64(3, 7)), dict(q_start=_i64(4)), dict(kv_len=_i64(3)), dict(mask=_i32(6, 4)), dict(mask=torch.zeros(6, 2, dtype=torch.float64).as_subclass(_OnDevice)),
                                    dict(q_start=_i32(3)), dict(kv_len=_i32(2)), dict(mask=_i64(5, 2)), dict(table=_i32(2, 7)), dict(table=_i32(20), table_stride=7),
                                    dict(table=_i32(3, 14)[:, ::2]), dict(kv_len=_i32(6)[::2]), dict(table=np.zeros((3, 7), np.int32)), dict(kv_len=torch.zeros(3, dtype=torch.int32))])
def test_tree_attention_refuses(library, change):
    with pytest.raises(ValueError):
        _tree(**change)
    assert not library.args


def test_the_table_may_be_a_slice(library):
    """Rows of a slice lie as far apart as those of what it is a slice of."""
    wide = _i32(5, 20)
    for table, stride in ((wide, 20), (wide[:, :7], 20), (wide[1:4, 3:10], 20), (wide[:3, :7].contiguous(), 7), (wide[::2, :8], 40)):
        _tree(table=table)
        assert (library.args[-1].table, library.args[-1].table_stride) == (table.data_ptr(), stride)
    one = wide[2:3, :7]  # (a single row: its length)
    R.tree_attention(R.F16, 1, 6, 4, 2, 64, 0x1000, 0x2000, 0x3000, 0x4000, one, 16, 30, _i32(2), _i32(1), 2, 7 * 16)
    assert library.args[-1].table_stride == 7


def test_rows_that_are_too_short_are_refused_by_the_library():
    """... and not read into what the slice leaves out."""
    wide = _i32(3, 20)
    with pytest.raises(R.R355Error) as e:
        R.tree_attention(R.F16, 3, 6, 4, 2, 64, 0x1000, 0x2000, 0x3000, 0x4000, wide[:, :7], 16, 30, _i32(4), _i32(3), 2, 8 * 16)
    assert e.value.code == -3


def test_zero_points(library):
    """... of the 4-bit products: bytes"""
    call = lambda zeros: R.w4_matmul(R.F16, R.F16, 4, 48, 200, 64, 0x1000, 0x2000, 0x3000, 0x4000, zeros=zeros)
    z = torch.zeros(4, 48, dtype=torch.uint8).as_subclass(_OnDevice)
    for zeros, address in ((z, z.data_ptr()), (None, None), (0x5000, 0x5000)):
        call(zeros)
        assert library.args[-1].zeros == address
    for zeros in (_i32(4, 48), _i64(4, 48), z[:3], z.t(), torch.zeros(4, 48, dtype=torch.uint8)):
        with pytest.raises(ValueError):
            call(zeros)
    assert len(library.args) == 3
