"""Where a position lies in a paged cache (paged.h, compiled for the host), and what the entry points that take one refuse.  Neither needs a GPU:
arguments are looked at before anything else."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import ane_amd.bridge as br

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ane_amd", "csrc")

PROGRAM = r"""
#include "paged.h"
#include <initializer_list>
#include <limits.h>
#include <stdio.h>
int main() {
    long n = 0;
    const int odd[] = {INT_MIN, INT_MIN + 1, -65536, -17, -1, 0, 1, 15, 16, 17, 47, 48, 1 << 20, INT_MAX - 1, INT_MAX};
    for (int page : {16, 48, 64, 65536})
        for (int n_seqs : {1, 3, INT_MAX})
            for (int max_pages : {1, 2, 5, INT_MAX})
                for (int seq : odd)
                    for (int pos : odd) {
                        const long long e = paged_entry(seq, pos, n_seqs, max_pages, page);
                        const bool in = seq >= 0 && seq < n_seqs && pos >= 0 && (long long)pos < (long long)max_pages * page;
                        if (in != (e >= 0)) return printf("entry of %d %d\n", seq, pos), 1;
                        if (in && e != (long long)seq * max_pages + pos / page) return printf("entry of %d %d is %lld\n", seq, pos, e), 1;
                        n++;
                    }
    for (int id : odd)
        for (int n_pages : {1, 16, INT_MAX}) {
            if (paged_id_ok(id, n_pages) != (id >= 0 && id < n_pages)) return printf("page %d of %d\n", id, n_pages), 1;
            n++;
        }
    // the last value of the largest page is inside, in 64 bits
    if (paged_row(INT_MAX - 1, 4095, 65535, 4096, 65536, 128) != ((size_t)(INT_MAX - 1) * 4096 + 4095) * 65536 * 128 + (size_t)65535 * 128) return puts("row"), 1;
    for (int page : {16, 48})
        for (int pos = -1; pos < 200; pos++)
            for (int parent = 0; parent < 2; parent++) {
                const PagedMove m = paged_move(1, parent, pos, page);
                if (pos < 0 ? m.moves || m.tail != -1 : m.tail != pos / page || m.filled != pos - m.tail * page + 1 || m.moves != (parent != 1 && m.filled < page))
                    return printf("move %d %d\n", parent, pos), 1;
                n++;
            }
    printf("%ld\n", n);
    return 0;
}
"""


def test_every_place(tmp_path):
    src, exe = tmp_path / "paged.cpp", tmp_path / "paged"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and int(out.stdout) > 1000, out.stdout


# Host memory stands for device memory: every call below is refused before it looks at any.
HOST = np.zeros(4096, np.float32)
P = (HOST.ctypes.data + 15) // 16 * 16


def cache(**over):
    c = dict(k=P, v=P, pages=P, n_pages=4, page=16, n_seqs=8, max_pages=2, kv_heads=2, hd=64)
    c.update(over)
    return br.KvCache(*c.values())


BAD_CACHES = [dict(k=None), dict(v=None), dict(pages=None), dict(n_pages=0), dict(page=0), dict(page=8), dict(page=24), dict(page=1 << 17), dict(page=-16),
              dict(n_seqs=0), dict(max_pages=0), dict(max_pages=-3), dict(max_pages=(1 << 26) + 1), dict(max_pages=2 ** 31 - 1), dict(kv_heads=0), dict(kv_heads=5000), dict(hd=0), dict(hd=4), dict(hd=60),
              dict(hd=136), dict(hd=-8), dict(k=P + 4), dict(v=P + 8)]


def refused(fn, *args):
    assert fn(*args) == -1 and br.last_error() and "usable" not in br.last_error(), (fn.__name__, br.last_error())


def names(stem):
    return [getattr(br.lib, "mi355_%s%s_dev" % (stem, e)) for e in ("", "_bf16")]


@pytest.mark.parametrize("fn", names("kv_append"))
def test_append_refuses(fn):
    ok = [cache(), P, P, P, P, P, P, P, P, 4, 4, 2, P, P, 100, 1e-6]
    def call(**over):
        a = list(ok)
        for i, v in over.items():
            a[int(i[1:])] = v
        if isinstance(a[0], br.KvCache):
            a[0] = C.byref(a[0])
        refused(fn, *a)
    for bad in BAD_CACHES:
        call(_0=cache(**bad))
    call(_0=None)
    for i in (3, 4, 8):
        call(**{"_%d" % i: None})
    call(_1=None), call(_2=None), call(_9=0)                                # q, q_out and heads
    call(_12=None), call(_13=None), call(_14=0), call(_14=-1)               # cos, sin and their table
    call(_9=3), call(_9=-2), call(_9=1 << 15), call(_10=0), call(_11=0), call(_10=1 << 22), call(_10=-1)
    call(_15=-1.0), call(_15=float("nan"))
    call(_7=None, _10=5)                                                    # ten columns, eight sequences
    call(_10=1 << 21, _9=64)                                                # more than a launch numbers


@pytest.mark.parametrize("fn", names("attn_paged"))
def test_attention_refuses(fn):
    ok = [cache(), P, P, P, P, P, 4, 4, 2, 0.125]
    def call(**over):
        a = list(ok)
        for i, v in over.items():
            a[int(i[1:])] = v
        if isinstance(a[0], br.KvCache):
            a[0] = C.byref(a[0])
        refused(fn, *a)
    for bad in BAD_CACHES:
        call(_0=cache(**bad))
    call(_0=None), call(_1=None), call(_3=None), call(_5=None)
    call(_6=0), call(_6=3), call(_6=-2), call(_6=1 << 15), call(_7=0), call(_8=0), call(_7=1 << 22)
    for scale in (0.0, -1.0, float("nan"), float("inf"), 3e38):
        call(_9=scale)
    call(_4=None, _7=5)
    call(_1=P, _3=P, _6=1 << 14, _7=1 << 11)
    call(_0=cache(page=1 << 16, max_pages=1 << 14, kv_heads=128), _6=128)       # more tiles than 32 bits count


@pytest.mark.parametrize("fn", names("beam_step"))
def test_beam_refuses(fn):
    q = P + 1024
    ok = [P, P, P, P, P, q, q, 100, 4, 2, 4, 2, 0]
    def call(**over):
        a = list(ok)
        for i, v in over.items():
            a[int(i[1:])] = v
        refused(fn, *a)
    for i in (0, 1, 2, 4, 5):
        call(**{"_%d" % i: None})
    call(_7=0), call(_8=0), call(_9=0), call(_10=0), call(_10=65, _8=65), call(_10=3), call(_8=1 << 22), call(_8=1 << 22, _9=1, _10=1), call(_7=1 << 30)
    call(_12=-1), call(_12=100), call(_11=100)
    call(_7=2**31 - 1, _10=1), call(_7=2**30 + 1, _10=1), call(_7=2**28 + 1)        # rows near 2^31: the places behind the last one would not fit 32 bits
    call(_0=q), call(_3=q)


@pytest.mark.parametrize("fn", names("kv_reorder"))
def test_reorder_refuses(fn):
    q = P + 1024
    def call(caches, count=None, **over):
        a = [(br.KvCache * len(caches))(*caches), len(caches) if count is None else count, q, q, q, P, P, P, 1]
        for i, v in over.items():
            a[int(i[1:])] = v
        refused(fn, *a)
    for bad in BAD_CACHES:
        call([cache(), cache(**bad)])
    for other in (dict(pages=P + 64), dict(n_pages=3), dict(page=32), dict(n_seqs=7), dict(max_pages=3), dict(kv_heads=1), dict(hd=72)):
        call([cache(), cache(**other)])
    call([cache()], count=0), call([cache()], count=-1)
    for i in (2, 4, 5, 6, 7):
        call([cache()], **{"_%d" % i: None})
    call([cache()], _2=P), call([cache()], _3=P), call([cache()], _4=P), call([cache()], _8=-1)
    call([cache(n_seqs=1 << 23)])
    refused(fn, None, 1, q, q, q, P, P, P, 1)
