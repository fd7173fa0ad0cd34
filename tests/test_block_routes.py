"""Which of the two attention kernels a call takes, by the library's own cost
rule: the batches that the tests make for the one or the other must go there,
or a change of the rule would leave a kernel untested."""
import os
import subprocess

import pytest

import lewm_b200 as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "le-wm-nv_b200", "lewm_b200")
MANY = 20000  # rows and new tokens of the batches that are meant for the tensor-core kernel
SOURCE = """
#include <cstdio>
#include <cstdlib>
#include "lwm_blocks.hpp"
int main(int argc, char** argv) {
    for (int i = 1; i + 10 < argc; i += 11) {
        const auto at = [&](int j) { return static_cast<uint32_t>(std::atol(argv[i + j])); };
        lwm::CacheAttnArgs a{};
        a.c.sequences = at(0), a.c.max_new = at(1), a.c.kv_heads = at(2), a.group = at(3), a.c.head_dim = at(4);
        a.c.table_stride = at(5), a.c.page_shift = at(6), a.c.max_length = at(7);
        a.window = at(8), a.sinks = at(9), a.frame = at(10), a.causal = 1;
        std::putchar(lwm::cache_attention_many_rows(a) ? '1' : '0');
    }
}
"""


@pytest.fixture(scope="module")
def many_rows(tmp_path_factory):
    at = tmp_path_factory.mktemp("routes")
    (at / "routes.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-I" + os.path.join(ROOT, "le-wm-nv_b200", "csrc"), "-I/usr/local/cuda/include",
                    str(at / "routes.cpp"), "-o", str(at / "routes"), os.path.join(LIB, os.path.basename(L.lib._name)),
                    "-Wl,-rpath," + LIB], check=True)

    def routes(calls):
        args = [str(x) for c in calls for x in c]
        out = subprocess.run([str(at / "routes"), *args], check=True, capture_output=True, text=True).stdout
        return [c == "1" for c in out]
    return routes


def call(sequences, new, kv, group, d, length, page=64, max_length=0, window=0, sinks=0, frame=1):
    return sequences, new, kv, group, d, -(-length // page), page.bit_length() - 1, max_length, window, sinks, frame


def test_padded_batches_take_the_tensor_core_kernel(many_rows):
    calls = [call(n, MANY, kv, group, d, length, page) for n in (1, 2, 3, 8) for kv, group in ((1, 1), (1, 3), (2, 1), (2, 4))
             for d in (32, 64, 128) for length, page in ((200, 64), (304, 16), (600, 32), (1025, 64))]
    calls += [call(6, MANY, 2, 3, d, 407, 32, window=w, sinks=s, frame=f) for d in (64, 128)
              for w, s, f in ((0, 0, 1), (0, 0, 7), (200, 1, 1), (1, 0, 197))]
    calls += [call(6, MANY, 2, 3, 32, 407, 32, frame=f) for f in (1, 7)]
    calls += [call(4, MANY, 1, 2, 64, 150, 16), call(3, MANY, 2, 2, 64, 96, 32), call(1, MANY, 8, 1, 128, 300, 128)]
    assert all(many_rows(calls))
    # windows of the tests that are there for masks at the edges of its tiles
    windows = [call(n, MANY, 1, 2, d, length, page, window=window, sinks=sinks) for n in (1, 2) for d in (32, 64, 128)
               for length, page in ((400, 32), (512, 32), (700, 64)) for window, sinks in ((150, 30), (160, 0), (180, 3), (160, 40))]
    assert all(many_rows(windows))


def test_few_rows_take_the_other_kernel(many_rows):
    calls = [call(n, new, kv, group, d, length) for n, kv, length in ((1, 1, 37), (3, 2, 300), (9, 2, 1030), (640, 1, 60),
                                                                      (1024, 16, 34), (2, 2, 5000), (48, 4, 30000))
             for new in (1, 3) for group in (1, 4) for d in (32, 64, 128)]
    assert not any(many_rows(calls))


def test_ordinary_calls_take_the_kernel_made_for_them(many_rows):
    whole, frames = call(2, 8192, 4, 4, 128, 8192), call(8, 394, 12, 1, 64, 7880, window=8, sinks=197, frame=197)
    token, chunk = call(4, 1, 8, 4, 128, 65536), call(1, 16, 8, 4, 128, 65536)
    assert many_rows([whole, frames, token, chunk]) == [True, True, False, False]
