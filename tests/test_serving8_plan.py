"""The sizes that the attention over an 8-bit cache lays its workspace out by, against the bytes that a caller is told to bring:
camelid_amd/csrc/paged8_plan.h, which the library is built from, compiled here and swept over sizes of calls."""
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "camelid_amd" / "csrc"

SWEEP = r"""
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>
#include "paged8_plan.h"
using namespace cm;
int main(int, char** v) {
  const uint32_t hd = (uint32_t)atoi(v[1]);
  const bool f32 = atoi(v[2]);
  std::mt19937_64 rng(hd + f32);
  const auto upto = [&](double most) {  // 1 .. most, spread over its logarithm
    return (uint64_t)std::exp2(std::uniform_real_distribution<double>(0, std::log2(most + 0.999))(rng));
  };
  uint64_t checked = 0, prompts = 0, cut = 0, bad = 0;
  const auto check = [&](size_t bytes, uint64_t n, uint64_t t, uint64_t nh, uint64_t n_kv, uint64_t cap) {
    const uint64_t g = nh / n_kv;
    if (n * n_kv > (1u << 20) || t * g * g >= (1ull << 32) || !grid_ok(n * n_kv * t * g, 256)) return;  // refused before
    const P8Sizes z = p8_sizes(n, t, nh, n_kv, hd, cap, f32);
    if (!z.fits) return;
    ++checked;
    prompts += z.prompt;
    cut += z.join;
    if (z.bytes <= bytes && z.part_o % 16 == 0 && z.cuts % 16 == 0 && z.part_o <= z.cuts && z.cuts <= z.bytes) return;
    if (!bad++) std::printf("n_seqs %zu n_new %zu n_heads %zu n_kv %zu cap %zu: %zu of %zu bytes\n", (size_t)n, (size_t)t,
                            (size_t)nh, (size_t)n_kv, (size_t)cap, z.bytes, bytes);
  };
  for (int i = 0; i < 100000; ++i) {
    const uint64_t g = upto(128), n_kv = upto(std::min(1024.0, 4096.0 / g)), nh = n_kv * g;
    const uint64_t n = upto(i % 2 ? 64 : 65535), t = i % 3 ? upto(300) : upto(1 << 20), cap = 16 * upto(1 << 20);
    const size_t bytes = p8_workspace(n, t, nh, n_kv, hd, cap);
    check(bytes, n, t, nh, n_kv, cap);
    for (int k = 0; k < 3; ++k) check(bytes, upto(n), upto(t), nh, n_kv, 16 * upto(cap / 16));
    // next to the borders between the kernels
    for (uint64_t near : {(uint64_t)8, (uint64_t)9, 127 / g, 128 / g + 1})
      if (near && near <= t) check(bytes, n, near, nh, n_kv, cap);
  }
  std::printf("%zu checked, %zu prompts, %zu cut, %zu bad\n", (size_t)checked, (size_t)prompts, (size_t)cut, (size_t)bad);
  return bad || checked < 100000 || prompts < checked / 20 || cut < checked / 20;
}
"""


@pytest.fixture(scope="module")
def sweep(tmp_path_factory):
    where = tmp_path_factory.mktemp("plan")
    (where / "sweep.cpp").write_text(SWEEP)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-I", str(CSRC), str(where / "sweep.cpp"), "-o",
                    str(where / "sweep")], check=True)
    return where / "sweep"


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("f32_rows", [0, 1])
def test_the_workspace_holds_its_layout(sweep, hd, f32_rows):
    run = subprocess.run([sweep, str(hd), str(f32_rows)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout
