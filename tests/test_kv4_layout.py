"""The 4-bit KV cache's layout (csrc/kernels/kv4_layout.hpp) on the CPU: every
code byte and scale of every row has a place of its own inside the head's
arrays, and the entry points refuse what they can see without a device."""
import ctypes as C
import os
import shutil
import subprocess
import sys

import pytest

import vlrf_amd as V
from vlrf_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "vlrf_amd/csrc/kernels/kv4_layout.hpp"
#include <cstdio>
#include <set>
using namespace vlrf_hip;
int main() {
    for (int d : {32, 64, 96, 128, 256})
        for (int seq : {1, 31, 32, 33, 200}) {
            std::set<size_t> k, v, s;
            for (int t = 0; t < seq; ++t) {
                if (kv4::key_of(kv4::lane_group(t), kv4::slot(t)) != t % 32) return 1;
                for (int b = 0; b < d / 32; ++b) {
                    s.insert(kv4::scale(t, b, d));
                    for (int i = 0; i < 16; ++i) {
                        k.insert(kv4::k_word(t, i / 4, b, d) + i % 4);
                        v.insert(kv4::v_byte(t, i, b, d));
                    }
                }
            }
            const size_t n = (size_t)seq * d / 2, m = (size_t)seq * d / 32;
            if (k.size() != n || v.size() != n || s.size() != m) return 2;
            if (*k.rbegin() >= kv4::head_codes(seq, d) || *v.rbegin() >= kv4::head_codes(seq, d)) return 3;
            if (*s.rbegin() >= kv4::head_scales(seq, d)) return 4;
        }
    // Past 32 bits: 100 million rows of 128.
    const int t = 99999999;
    if (kv4::k_word(t, 3, 3, 128) != (size_t)t * 64 + 60 || kv4::k_word(t, 3, 3, 128) >= kv4::head_codes(t + 1, 128)) return 5;
    if (kv4::v_byte(t, 15, 3, 128) >= kv4::head_codes(t + 1, 128) || kv4::v_byte(t, 15, 3, 128) < ((size_t)5 << 30)) return 6;
    if (kv4::scale(t, 3, 128) >= kv4::head_scales(t + 1, 128)) return 7;
    return 0;
}
"""


def test_every_code_and_scale_has_its_own_place(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    src, exe = tmp_path / "layout.cpp", tmp_path / "layout"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", ROOT, str(src), "-o", str(exe)], check=True, timeout=120)
    assert subprocess.run([str(exe)], timeout=60).returncode == 0


def test_null_handles_are_refused():
    lib, x = V.lib(), C.c_void_p(16)
    assert V.KV_Q4_0 == 3
    assert lib.vlrf_hip_kv_truncate(None, 0, 0) == _lib.ERR_ARG and "null cache" in _lib.last_error()
    assert lib.vlrf_hip_attn_chunk(None, 0, x, x, 1, 1, 1, 1.0) == _lib.ERR_ARG and "null cache" in _lib.last_error()
    h = C.c_void_p()
    assert lib.vlrf_hip_kv_create(None, 1, 1, 1, 64, V.KV_Q4_0, C.byref(h)) == _lib.ERR_ARG and h.value is None


def test_scratch_of_refused_attention_is_none():
    """The scratch of an attention is asked for before the launch refuses its sizes: none for those, any
    d_head that a cache may have. In a process of its own: a division by no rows would end it."""
    code = ("import sys; sys.path.insert(0, %r)\n"
            "import ctypes as C\n"
            "import vlrf_amd as V\n"
            "part = V.lib()._ZN8vlrf_hip19attn_kv4_part_bytesEiiiii\n"
            "part.restype, part.argtypes = C.c_size_t, [C.c_int] * 5\n"
            "for d in (32, 96, 160, 256, 512, 544, 1024, 65536):\n"
            "    for H, G, T, n in ((4, 1, 1, 100), (32, 8, 1, 120001), (32, 8, 40, 3001), (32, 8, 1777, 4001)):\n"
            "        assert part(H, G, d, T, n) == 0, (H, G, d, T, n)\n"
            "for H, G, T, n in ((0, 1, 1, 9000), (4, 0, 1, 9000), (4, 3, 1, 9000), (-4, 1, 1, 9000), (4, 1, 0, 9000), (4, 1, 9, 8)):\n"
            "    assert part(H, G, 64, T, n) == 0, (H, G, T, n)\n"
            "assert part(32, 8, 128, 1, 120001) == 32 * 32 * 132 * 4 and part(32, 4, 64, 1, 100) == 0\n"
            "print('ok')" % ROOT)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", (r.returncode, r.stderr[-800:])


def test_fixed_scratch_serves_long_contexts():
    """What a decode row's partials need beside the 2^19 floats of the call that allocates nothing: less at
    any context with up to 15 query heads a KV head or heads of 64."""
    part = V.lib()._ZN8vlrf_hip19attn_kv4_part_bytesEiiiii
    part.restype, part.argtypes = C.c_size_t, [C.c_int] * 5
    for d in (64, 128):
        for G in (1, 2, 3, 4, 8, 16, 40):
            for rep in range(1, 41):
                for n in (1, 256, 257, 8065, 20000, 65536, 65537, 120001, 1 << 20, 1 << 27):
                    need = part(G * rep, G, d, 1, n) // 4
                    assert need <= 256 * 16 * (d + 4)
                    if d == 64 or rep < 16:
                        assert need <= 1 << 19, (G, rep, d, n)
    for H, G, n in ((16, 1, 65536), (128, 8, 8192)):
        assert part(H, G, 128, 1, n) // 4 <= 1 << 19 < part(H, G, 128, 1, n + 1) // 4
