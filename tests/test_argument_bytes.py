"""The argument structures that Python writes as bytes against what the compiler makes of the header."""
import ctypes
import os
import subprocess

import rocwmma_amd as R

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "r355_wmma.h")
PART = ["x", "y", "heads", "rotate", "to_slots", None, "x_token_stride", "x_head_stride", "y_token_stride", "y_head_stride"]
ROPE = (["type", "layout", "tokens", "head_dim", "rotary_dim", "parts"] + [f and "part[%d].%s" % (i, f) for i in range(3) for f in PART]
        + ["positions", "turns", "slots", "slot_count", "inverse", "scale"])
TREE = ["type", "batch", "total_tokens", "heads", "kv_heads", "head_dim", "max_tokens", "max_kv", "q", "k", "v", "out", "lse", "q_token_stride", "q_head_stride", "k_slot_stride",
        "k_head_stride", "v_slot_stride", "v_head_stride", "out_token_stride", "out_head_stride", "table", "table_stride", "page_size", "pages", None, "q_start", "kv_len", "mask",
        "mask_words", None, "scale", "workspace", "workspace_bytes"]


def _layout(tmp_path, name, fields):
    """{field: (offset, size)} of a structure of the header, and its size"""
    rows = "".join('    printf("%%zu %%zu\\n", offsetof(%s, %s), sizeof(((%s*)0)->%s));\n' % (name, f, name, f) for f in fields)
    source, program = str(tmp_path / "layout.c"), str(tmp_path / "layout")
    with open(source, "w") as out:
        out.write('#include <stddef.h>\n#include <stdio.h>\n#include "%s"\nint main(void)\n{\n%s    printf("%%zu\\n", sizeof(%s));\n    return 0;\n}\n' % (HEADER, rows, name))
    subprocess.check_call(["gcc", "-o", program, source])
    lines = subprocess.check_output([program], text=True).split("\n")
    return {f: tuple(int(n) for n in line.split()) for f, line in zip(fields, lines)}, int(lines[len(fields)])


def _check(packed, names, tmp_path, name):
    """Every field of the bytes, made one at a time not zero, lies where the header has it."""
    layout, size = _layout(tmp_path, name, [n for n in names if n])
    assert packed.size == size
    letters = [c for c in _letters(packed.format)]
    assert len(letters) == len(names)
    for i, (field, letter) in enumerate(zip(names, letters)):
        values = [0.0 if c == "d" else 0 for c in letters]
        values[i] = -1.0 if letter == "d" else -1 if letter in "iq" else {"I": 2 ** 32 - 1, "Q": 2 ** 64 - 1}[letter]
        at = [j for j, byte in enumerate(packed.pack(*values)) if byte]
        if field:
            offset, length = layout[field]
            assert at and offset <= at[0] and at[-1] < offset + length and ({"i": 4, "I": 4, "q": 8, "Q": 8, "d": 8}[letter] == length), field
        else:
            assert all(not o <= at[0] < o + n for o, n in layout.values())


def _letters(text):
    return text.lstrip("=")


def test_rope_args(tmp_path):
    _check(R._ROPE_ARGS, ROPE, tmp_path, "r355_rope_args")


def test_tree_attention_args(tmp_path):
    _check(R._TREE_ARGS, TREE, tmp_path, "r355_tree_attention_args")
    assert ctypes.sizeof(R.TreeAttentionArgs) == R._TREE_ARGS.size
    names = [n for n in TREE if n]
    assert [f for f, _ in R.TreeAttentionArgs._fields_] == names
    layout, _ = _layout(tmp_path, "r355_tree_attention_args", names)
    assert {n: (getattr(R.TreeAttentionArgs, n).offset, getattr(R.TreeAttentionArgs, n).size) for n in names} == layout


def test_w4_args(tmp_path):
    names = [f for f, _ in R.W4Args._fields_]
    layout, size = _layout(tmp_path, "r355_w4_args", names)
    assert ctypes.sizeof(R.W4Args) == size
    assert {n: (getattr(R.W4Args, n).offset, getattr(R.W4Args, n).size) for n in names} == layout
