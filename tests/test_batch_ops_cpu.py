"""The operators of a batched step without a GPU: the caches and batches that the calls refuse, the
scratch they ask for, and the tests' own step-by-step pages (no device is touched)."""
import ctypes as C

import numpy as np
import pytest

from batch_ops_ref import Pages
from charsiu_b200 import lib as L

BF16 = 30


def cache(**changes):
    p = L.PagesStruct(k=1 << 20, v=1 << 21, table=1 << 12, len=1 << 12, ref=1 << 12, work=1 << 12,
                      layer_stride=1 << 16, page_stride=8192, pos_stride=512, head_stride=64,
                      type=BF16, n_layer=2, n_pages=8, page=16, n_head_kv=8, head_dim=64, n_seq=4,
                      max_pages=4)
    for k, v in changes.items():
        setattr(p, k, v)
    return p


def work(p):
    return L.lib().charsiu_gpu_pages_work(C.byref(p))


def test_a_good_cache_has_scratch():
    assert work(cache()) >= 4 * 8
    assert work(cache(n_pages=1000)) > work(cache())


@pytest.mark.parametrize("changes", [
    dict(k=None), dict(v=None), dict(table=None), dict(len=None), dict(ref=None), dict(type=0),
    dict(type=8), dict(page=0), dict(page=8), dict(page=24), dict(page=256), dict(head_dim=32),
    dict(head_dim=96), dict(n_layer=0), dict(n_pages=0), dict(n_head_kv=0), dict(n_seq=0),
    dict(max_pages=0), dict(k=(1 << 20) + 8), dict(v=(1 << 20) + 2), dict(table=(1 << 12) + 2),
    dict(layer_stride=4), dict(page_stride=8190), dict(pos_stride=68), dict(head_stride=1),
    dict(pos_stride=56), dict(head_stride=0), dict(n_pages=(1 << 21) + 1), dict(max_pages=1 << 28)],
    ids=str)
def test_bad_caches_are_refused(changes):
    assert work(cache(**changes)) == 0


def test_no_layer_no_call():
    lib = L.lib()
    p, b = cache(), L.AttentionStruct()
    s = (L.AdaptersStruct * 1)()
    assert lib.charsiu_gpu_norm_quantise_dev(None, 1, None, 1, 1, 32, 1e-5, None, 1, 1, None) == -1
    assert lib.charsiu_gpu_pages_grow_dev(None, C.byref(p), 1, 1, 1, None) == -1
    assert lib.charsiu_gpu_pages_fork_dev(None, C.byref(p), 1, 1, 1, None) == -1
    assert lib.charsiu_gpu_pages_free_dev(None, C.byref(p), 1, 1, None) == -1
    assert lib.charsiu_gpu_pages_compact_dev(None, C.byref(p), None, None) == -1
    assert lib.charsiu_gpu_pages_append_dev(None, C.byref(p), 0, 1, 1, 1, 8, 1, 1, 1, 1, 1, 1,
                                            None) == -1
    assert lib.charsiu_gpu_attention_work(None, C.byref(p), C.byref(b)) == 0
    assert lib.charsiu_gpu_attention_dev(None, C.byref(p), 0, C.byref(b), 1, 1, None) == -1
    assert lib.charsiu_gpu_adapters_work(None, s, 1, 1) == 0
    assert lib.charsiu_gpu_adapters_dev(None, s, 1, 1, 1, 1, 1, None, None, None, 0, None) == -1


def test_struct_sizes(tmp_path):
    """The ctypes mirrors are the header's structs."""
    import os
    import subprocess
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "charsiu_gpu.h"\nint main(void) { printf("%zu %zu %zu\\n", '
                   "sizeof(struct charsiu_gpu_pages), sizeof(struct charsiu_gpu_attention), "
                   "sizeof(struct charsiu_gpu_adapters)); return 0; }\n")
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c11", f"-I{inc}", str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == [C.sizeof(L.PagesStruct), C.sizeof(L.AttentionStruct),
                                     C.sizeof(L.AdaptersStruct)]


def test_the_plain_pages_keep_their_books():
    """References count the slots that hold a page, through grows, forks, frees and packing."""
    rng = np.random.default_rng(5)
    p = Pages(np.zeros((6, 5), np.int32), np.zeros(6, np.int32), np.zeros(16, np.int32),
              rng.standard_normal((1, 16, 4, 1, 2)), rng.standard_normal((1, 16, 4, 1, 2)), 4)

    def check():
        held = np.zeros(16, int)
        for s, n in enumerate(p.len):
            for j in range(-(-n // 4)):
                held[p.table[s, j]] += 1
        assert np.array_equal(held, p.ref)

    for _ in range(200):
        what, a, b = rng.integers(4), rng.integers(6, size=3), rng.integers(6, size=3)
        if what == 0:
            p.grow(list(a), int(rng.integers(1, 9)))
        elif what == 1:
            p.fork(list(a), list(b))
        elif what == 2:
            p.free(list(a[:2]))
        else:
            assert p.compact() == (p.ref > 0).sum() and not p.ref[(p.ref > 0).sum():].any()
        check()
    assert p.refused > 0


def run_check(tmp_path, name):
    """tests/<name>.cpp against the headers it includes."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = str(tmp_path / name)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", f"-I{root}/include", f"-I{root}/charsiu_b200/csrc",
                    f"{root}/tests/{name}.cpp", "-o", exe], check=True)
    got = subprocess.run([exe], capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout.startswith("ok "), got.stdout


def test_the_checks_of_sizes_and_pointers(tmp_path):
    """batch_checks.h by itself: sizes whose product passes 64 bits among them."""
    run_check(tmp_path, "batch_checks_check")


def test_the_cuts_of_the_longest_sequences(tmp_path):
    """attn_cut.h by itself, up to the longest length that a cache may tell."""
    run_check(tmp_path, "attn_cut_check")
