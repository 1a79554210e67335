"""The layer loop's attention operators without a GPU: refusals that come before a device is touched,
struct layouts, and the cache's addressing, from the library's own header compiled here: every value of
every token has a place of its own inside its record, and the last record of caches past 4 GiB ends
inside the allocation."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

import layer_util as L
import turbo_decode_tail as T

CSRC = Path(__file__).resolve().parents[1] / "turbo-winfare_amd" / "csrc"
PROGRAM = """
#include <cstdio>
#include <vector>
#include "dt_kv.h"
using namespace tdt;
int main() {
    for (uint32_t groups : {1u, 2u, 4u, 8u}) for (uint32_t bits : {4u, 8u}) {
        const uint32_t d = groups * 64u, part = kv_part_bytes(groups, bits), rec = kv_record_bytes(groups, bits);
        if (part != d * 32u * bits / 8u || rec != 2u * part + 2u * groups * 128u) return 1;
        std::vector<int> key(2u * part), value(2u * part), scale((rec - 2u * part) / 4u);  // by half bytes
        for (uint32_t t = 0; t < 32u; ++t) for (uint32_t e = 0; e < d; ++e) {
            const uint32_t kb = kv_key_byte(bits, t, e), vb = kv_value_byte(bits, t, e);
            if (kb >= part || vb >= part) return 2;
            if (bits == 8u) ++key[2u * kb], ++key[2u * kb + 1u], ++value[2u * vb], ++value[2u * vb + 1u];
            else ++key[2u * kb + (e & 1u)], ++value[2u * vb + ((e >> 4) & 1u)];
            // four tokens in a row from a multiple of four on are neighbouring bytes of the values
            if (t % 4u == 0u) for (uint32_t j = 0; j < 4u; ++j) if (kv_value_byte(bits, t + j, e) != vb + j || vb % 4u) return 3;
        }
        for (uint32_t i = 0; i < 2u * part; ++i) if (key[i] != 1 || value[i] != 1) return 4;
        for (uint32_t w = 0; w < 2u; ++w) for (uint32_t t = 0; t < 32u; ++t) for (uint32_t g = 0; g < groups; ++g) {
            const uint32_t at = kv_scale_byte(groups, w, t, g);
            if (at % 4u || at + 4u > rec - 2u * part) return 5;
            ++scale[at / 4u];
        }
        for (int n : scale) if (n != 1) return 6;
        for (uint32_t shift : {5u, 8u}) for (uint32_t heads : {1u, 8u, 1024u}) for (uint64_t slots : {64ull, 4000000000ull}) {
            KvView kv{};
            kv.page_shift = shift, kv.heads = heads, kv.bits = bits, kv.groups = groups, kv.record = rec;
            kv.pages = (uint32_t)(slots >> shift) + 1u;
            const unsigned __int128 want = (unsigned __int128)kv.pages * heads * ((1u << shift) / 32u) * rec;
            if (want >> 63) continue;
            const uint64_t bytes = kv_record_at(kv, kv.pages, 0, 0);
            if (bytes != (uint64_t)want) return 7;
            if (kv_record_at(kv, kv.pages - 1u, heads - 1u, (1u << shift) / 32u - 1u) + rec != bytes) return 8;
        }
    }
    return 0;
}
"""


def test_every_value_has_its_place(tmp_path):
    (tmp_path / "kv.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++20", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{CSRC}", str(tmp_path / "kv.cpp"),
                    "-o", str(tmp_path / "kv")], check=True)
    assert subprocess.run([str(tmp_path / "kv")]).returncode == 0


def test_a_grid_holds_fewer_than_two_to_the_32_threads(tmp_path):
    (tmp_path / "grid.cpp").write_text("""
#include "dt_kv.h"
bool refused(uint64_t n) { try { return tdt::grid_blocks(n) != n; } catch (const std::runtime_error&) { return true; } }
int main() { return refused(1) || refused((1u << 24) - 1u) || !refused(1u << 24) || !refused(1ull << 32) || !refused((1ull << 32) + 5u); }
""")
    subprocess.run(["g++", "-std=c++20", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{CSRC}", str(tmp_path / "grid.cpp"),
                    "-o", str(tmp_path / "grid")], check=True)
    assert subprocess.run([str(tmp_path / "grid")]).returncode == 0


def test_struct_sizes():
    lib = T.load()
    for which, st in ((6, T.TurboKvCacheDesc), (7, T.TurboRotaryDesc), (8, T.TurboQkvInputs), (9, T.TurboAttentionInputs)):
        assert lib.turbo_abi_struct_size(which) == C.sizeof(st), st.__name__


@pytest.mark.parametrize("field,value,word", [("head_dim", 96, "head_dim"), ("head_dim", 0, "head_dim"), ("bits", 5, "bits"),
                                              ("page_tokens", 48, "page_tokens"), ("page_tokens", 512, "page_tokens"),
                                              ("kv_heads", 0, "kv_heads"), ("kv_heads", 1025, "kv_heads"), ("pages", 0, "pages"),
                                              ("pages", 2**31, "2^32")])
def test_cache_refuses(field, value, word):
    lib = T.load()
    d = T.TurboKvCacheDesc()
    lib.turbo_kv_cache_desc_default(C.byref(d))
    d.pages = 4
    setattr(d, field, value)
    assert not lib.turbo_kv_cache_create(C.byref(d))
    assert word in T.last_error()


@pytest.mark.parametrize("field,value,word", [("head_dim", 80, "head_dim"), ("rotary_dim", 258, "rotary_dim"),
                                              ("rotary_dim", 24, "rotary_dim"), ("layout", 2, "layout"), ("norms", 8, "norms"),
                                              ("eps", -1.0, "eps"), ("eps", float("nan"), "eps"), ("theta", 0.0, "theta"),
                                              ("theta", float("inf"), "theta")])
def test_rotary_refuses(field, value, word):
    lib = T.load()
    d = T.TurboRotaryDesc()
    lib.turbo_rotary_desc_default(C.byref(d))
    setattr(d, field, value)
    assert not lib.turbo_rotary_create(C.byref(d))
    assert word in T.last_error()


def test_rotary_refuses_a_frequency_that_is_not_finite():
    with pytest.raises(T.TurboError, match=r"inv_freq\[3\]"):
        T.Rotary(64, inv_freq=[1.0] * 3 + [float("nan")] + [0.0] * 28)


def test_null_handles():
    lib = T.load()
    lib.turbo_kv_cache_destroy(None)
    lib.turbo_rotary_destroy(None)
    assert lib.turbo_kv_cache_write(None, None, 0, None, 0, 0, None, 1, None) == 0 and "handle" in T.last_error()
    assert lib.turbo_kv_cache_read(None, None, 1, 0, None, 0, None, 0, None) == 0 and "handle" in T.last_error()
    assert lib.turbo_qk_norm_rope(None, None, None) == 0 and "handle" in T.last_error()
    assert lib.turbo_prefix_attention(None, None, None) == 0 and "handle" in T.last_error()
    assert lib.turbo_attention_workspace(None, None, None) == 0 and "handle" in T.last_error()
    assert not lib.turbo_kv_cache_create(None) and not lib.turbo_rotary_create(None)


def test_plain_quantiser():
    """The tests' own quantiser keeps its definition: every value within half a step, the ends covered."""
    rng = np.random.default_rng(1)
    for bits in (4, 8):
        x = (rng.standard_normal((50, 128)) * 10.0 ** rng.integers(-6, 6, (50, 1))).astype(np.float32)
        x[0], x[1, :64], x[2] = 0.0, -7.25, np.float32(-0.0)
        c, s, b = L.quantise(x, bits)
        back = L.stored(x, bits)
        assert np.all(np.abs(back - x) <= np.repeat(s, 64, axis=1) * (0.5 + 2.0**-15))
        assert np.all(b <= x.reshape(50, 2, 64).min(-1)) and np.all(L.bf16(s) == s) and np.all(L.bf16(b) == b)
        assert c.max() == 2**bits - 1 and np.all(back[0] == 0.0) and np.all(back[1, :64] == -7.25)
