"""What a part of a rotation keeps between rope_part() and rope() (on the CPU: the address of host memory is as good as any where nothing is launched)."""
import weakref

import pytest
import torch

import rocwmma_amd as R


def test_a_part_keeps_its_tensors():
    """A tensor that only the part knows must not be freed before the call, or the next one that is made may get its memory."""
    x, y = (torch.zeros(4, 2, 64, dtype=torch.float16) for _ in range(2))
    refs = weakref.ref(x), weakref.ref(y)
    part = R.rope_part(x, y, 2, (128, 64), (128, 64))
    del x, y
    assert all(r() is not None for r in refs)
    del part
    assert all(r() is None for r in refs)


def test_parts_are_read_in_their_order(monkeypatch):
    seen = []

    class Library:
        def r355_rope(self, args, stream):
            seen.append(R._ROPE_ARGS.unpack(args))
            return 0

    monkeypatch.setattr(R, "lib", Library)
    tensors = [torch.zeros(4, h, 64) for h in (3, 2, 1)]
    parts = [R.rope_part(t, t, t.shape[1], (64 * t.shape[1], 64), (7 + i, 8 + i), rotate=i < 2, to_slots=i > 0) for i, t in enumerate(tensors)]
    for n in (1, 2, 3):
        R.rope(R.F32, R.ROPE_INTERLEAVED, 4, 64, 32, parts[:n], 0x3000, 0x4000, scale=1.5, inverse=True, slots=0x5000, slot_count=9)
        fields = seen[-1]
        assert fields[:6] == (R.F32, R.ROPE_INTERLEAVED, 4, 64, 32, n)
        for i in range(3):
            t = tensors[i]
            want = (t.data_ptr(), t.data_ptr(), t.shape[1], i < 2, i > 0, 0, 64 * t.shape[1], 64, 7 + i, 8 + i) if i < n else (0,) * 10
            assert fields[6 + 10 * i: 16 + 10 * i] == want
        assert fields[36:] == (0x3000, 0x4000, 0x5000, 9, 1, 1.5)


def test_no_part_and_four_parts_are_refused():
    part = R.rope_part(0x1000, 0x2000, 2, (128, 64), (128, 64))
    for n in (0, 4):
        with pytest.raises(ValueError):
            R.rope(R.F16, R.ROPE_HALF, 4, 64, 64, [part] * n, 0x3000, 0x4000)
