"""Drafted-tree and sampling entry points without a GPU: argument checks that come before the
device, and the ctypes mirrors of their structs."""
import ctypes as C
import importlib
import subprocess
from pathlib import Path

import pytest

L = importlib.import_module("gemma4-js_b200._lib")
P = C.c_void_p(4096)  # a non-null pointer that no refused call touches


def refused(name, *args):
    st = getattr(L.load(), name)(*args)
    return st, L.load().g4_last_error_string().decode()


def how(uniform=4096):
    return C.byref(L.G4Sampling(None, None, None, None, uniform))


@pytest.mark.parametrize("args,status,text", [
    ((P, 10, -1, 10, 0.0, how(), P, P), -1, "rows"),
    ((P, 9, 1, 10, 0.0, how(), P, P), -1, "pitch"),
    ((P, 10, 1, 0, 0.0, how(), P, P), -1, "vocab"),
    ((P, 800000, 1, 786433, 0.0, how(), P, P), -5, "786432"),
    ((P, 10, 1, 10, 0.0, None, P, P), -1, "g4_sample"),
    ((P, 10, 1, 10, 0.0, how(None), P, P), -1, "null"),
    ((None, 10, 1, 10, 0.0, how(), P, P), -1, "null"),
    ((P, 10, 1, 10, 0.0, how(), None, P), -1, "null"),
    ((P, 10, 1, 10, 0.0, how(), P, None), -1, "null context"),  # all in order but the context
])
def test_sample_arguments(args, status, text):
    st, msg = refused("g4_sample", None, *args)
    assert st == status and text in msg


def tree(nodes=4, stride=4, parents=4096):
    return C.byref(L.G4Tree(parents, stride, nodes, None))


def rows(n=4, pos=4096, base=0):
    return C.byref(L.G4Rows(pos, base, n, 0, 0))


@pytest.mark.parametrize("args,status,text", [
    ((P, None, 4, 8, 256, rows(), tree(65), 100, 0, 0, P), -5, "64"),
    ((P, None, 4, 8, 256, rows(), tree(0), 100, 0, 0, P), -5, "nodes"),
    ((P, None, 4, 8, 256, rows(), tree(parents=None), 100, 0, 0, P), -1, "null tree"),
    ((P, None, 4, 8, 256, rows(), None, 100, 0, 0, P), -1, "null tree"),
    ((P, None, 4, 8, 256, rows(), tree(stride=3), 100, 0, 0, P), -1, "parent_stride"),
    ((P, None, 4, 8, 256, rows(3), tree(), 100, 0, 0, P), -1, "rows per sequence"),
    ((P, None, 4, 8, 256, rows(pos=None), tree(), 100, 0, 0, P), -1, "positions"),
    ((P, None, 4, 8, 256, None, tree(), 100, 0, 0, P), -1, "map"),
    ((P, None, 6, 8, 256, rows(), tree(), 100, 0, 0, P), -1, "multiple"),
    ((P, None, 4, 8, 256, rows(base=-1), tree(), 100, 0, 0, P), -1, "seq_base"),
    ((P, None, 4, 9, 256, rows(), tree(), 100, 0, 0, P), -5, "heads"),
    ((P, None, 4, 8, 256, rows(), tree(), 100, 1, 0, P), -1, "window"),
    ((C.c_void_p(4098), None, 4, 8, 256, rows(), tree(), 100, 0, 0, P), -1, "aligned"),
    ((P, None, 4, 8, 256, rows(), tree(), 100, 0, 0, P), -1, "null argument"),
])
def test_attention_tree_arguments(args, status, text):
    st, msg = refused("g4_attention_tree", None, *args)
    assert st == status and text in msg


def test_row_mover_arguments():
    kv = (C.c_void_p * 1)(4096)
    ints = lambda *v: (C.c_int32 * len(v))(*v)  # noqa: E731
    assert refused("g4_tree_accept", None, tree(), -1, P, P, P, P, P)[0] == -1
    assert refused("g4_tree_accept", None, tree(70), 1, P, P, P, P, P)[0] == -5
    assert refused("g4_tree_accept", None, tree(), 1, P, None, P, P, P)[0] == -1
    assert "null context" in refused("g4_tree_accept", None, tree(), 1, P, P, P, P, P)[1]
    assert refused("g4_kv_compact", None, kv, 1, 10, P, 0, 1, 65, P, P)[0] == -5
    assert refused("g4_kv_compact", None, kv, 1, 10, None, 0, 1, 4, P, P)[0] == -1
    assert refused("g4_kv_compact", None, kv, 1, 10, P, -1, 1, 4, P, P)[0] == -1
    assert "source and a destination" in refused("g4_kv_fork", None, kv, 1, 10, P, ints(0, 1), ints(1, 2), 2)[1]
    assert "twice" in refused("g4_kv_fork", None, kv, 1, 10, P, ints(0, 1), ints(3, 3), 2)[1]
    assert refused("g4_kv_fork", None, kv, 1, 10, P, ints(-1), ints(3), 1)[0] == -6
    assert refused("g4_kv_fork", None, kv, 1, 10, P, None, None, 1)[0] == -1
    assert "null context" in refused("g4_kv_fork", None, kv, 1, 10, P, ints(0), ints(3), 1)[1]
    assert refused("g4_advance_positions_each", None, P, 0, 1, None)[0] == -1
    y = C.byref(L.G4Planes(4096, 1, 0, 100))
    assert refused("g4_qkv_post_tree", None, y, 8, 256, P, P, 1e-6, 0, 1e4, rows(3), tree(), 4, P, None, 0)[0] == -1
    assert refused("g4_qkv_post_tree", None, y, 0, 256, P, P, 1e-6, 0, 1e4, rows(), tree(), 4, P, None, 0)[0] == -1


def test_struct_layouts_match_the_header(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text(
        '#include <stddef.h>\n#include <stdio.h>\n#include "g4w4.h"\n'
        'int main(void) { printf("%zu %zu %zu %zu %zu %zu %zu %d\\n", sizeof(g4_sampling), offsetof(g4_sampling, top_k),\n'
        "  offsetof(g4_sampling, uniform), sizeof(g4_tree), offsetof(g4_tree, parent_stride), offsetof(g4_tree, nodes),\n"
        "  offsetof(g4_tree, counts), G4_TREE_MAX_NODES); return 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-I", str(Path(L.HEADER).parent), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    S, T = L.G4Sampling, L.G4Tree
    assert got == [C.sizeof(S), S.top_k.offset, S.uniform.offset, C.sizeof(T), T.parent_stride.offset, T.nodes.offset,
                   T.counts.offset, L.G4_TREE_MAX_NODES]
