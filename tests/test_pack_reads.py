"""The copy of odd operands reads four values at a time from rows that start anywhere: through types that are aligned to one
value.  Built for the host, where the compiler's alignment check ends a program that reads by more than its type is aligned to."""
import subprocess

import pytest

import mfma_hazards  # noqa: F401  (puts build_lib on the path)
from build_lib import HIPFLAGS, _hipcc

PROGRAM = r"""
#include "gdn2_linear.hpp"
#include <cstdio>
#include <vector>
int main() {
  std::vector<uint32_t> store(64);
  for (int lead = 0; lead < 8; ++lead) {
    uint32_t v[4];
    uint16_t* half = reinterpret_cast<uint16_t*>(store.data()) + lead;
    for (int i = 0; i < 12; ++i) half[i] = (uint16_t)(0x8000u + 257u * i);
    for (int at = 0; at < 5; ++at) {
      gdn2::lin_four<false>(half, at, v);
      for (int e = 0; e < 4; ++e)
        if (v[e] != half[at + e]) return 1;
    }
    uint32_t* whole = store.data() + 16 + lead;
    for (int i = 0; i < 12; ++i) whole[i] = 0x80000001u + 16777259u * i;
    for (int at = 0; at < 5; ++at) {
      gdn2::lin_four<true>(whole, at, v);
      for (int e = 0; e < 4; ++e)
        if (v[e] != whole[at + e]) return 2;
    }
  }
  std::puts("read");
}
"""


def test_four_values_from_any_place(tmp_path):
    src, exe = tmp_path / "reads.hip", tmp_path / "reads"
    src.write_text(PROGRAM)
    flags = [f for f in HIPFLAGS if f != "-O3"]
    r = subprocess.run([_hipcc(), *flags, "-O1", "-w", "-I" + str(mfma_hazards.PKG / "csrc"), "--cuda-host-only", "-Xarch_host",
                        "-fsanitize=alignment", "-Xarch_host", "-fsanitize-trap=alignment", str(src), "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "read\n", (r.returncode, r.stderr[-500:])


@pytest.mark.gpu
@pytest.mark.parametrize("lead", [1, 3, 4])
@pytest.mark.parametrize("stride", [517, 519, 520])
def test_operands_that_are_copied(stride, lead):
    """Rows of odd strides and starts, in the types whose operands are copied, against sums in 64 bits (2000 x 1000 results:
    the bound of a sum of K = 515 products in float32, (K / 32 + 12) 2^-22 of the absolute ones, and half a step)."""
    import torch
    from atomic_gdn2.linear import linear
    gen = torch.Generator(device="cuda").manual_seed(stride + lead)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        x = torch.randn((2000, stride + lead), device="cuda", generator=gen).to(dt)[:, lead:lead + 515]
        w = torch.randn((515, 1101 + lead), device="cuda", generator=gen).to(dt)[:, lead:lead + 1000]
        y = linear(x, w).double()
        X, W = x.double(), w.double()
        bound = (515 / 32 + 12) * 2.0 ** -22 * (X.abs() @ W.abs()) + torch.finfo(dt).eps / 2 * (X @ W).abs() + 1e-30
        assert ((y - X @ W).abs() <= bound).all()
