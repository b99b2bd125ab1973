"""A kernel's attributes belong to a device: they are set on every one that it is launched on (csrc/per_device.h)."""
import re
import subprocess
from pathlib import Path

import pytest
import torch

from tyr_b200.ops import _common
from tyr_b200.ops.paged_cache import PagedStore, paged_append, paged_attention
from tyr_b200.ops.sampling import sample

CSRC = Path(__file__).resolve().parents[1] / "csrc"

PROGRAM = r"""
#include <cstdio>
#include "per_device.h"
int main() {
  tyr::OncePerDevice ready;
  int calls = 0, fails = 1;
  auto set = [&] { ++calls; return fails > 0 ? fails-- : 0; };
  const int first = ready(0, set), again = ready(0, set), kept = ready(0, set), second = ready(1, set), kept2 = ready(1, set), last = ready(63, set), kept63 = ready(63, set);
  const int far = ready(64, set), far2 = ready(64, set);
  std::printf("%d %d %d %d %d %d %d %d %d %d\n", first, again, kept, second, kept2, last, kept63, far, far2, calls);
}
"""


def test_every_device_is_set_up_once_and_failures_are_tried_again(tmp_path):
    (tmp_path / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", str(CSRC), str(tmp_path / "main.cpp"), "-o", str(tmp_path / "main")], check=True)
    # one failure, then devices 0, 1 and 63 once each, and number 64 at both calls
    assert subprocess.run([str(tmp_path / "main")], capture_output=True, text=True, check=True).stdout.split() == "1 0 0 0 0 0 0 0 0 6".split()


def test_no_unit_sets_attributes_once_for_the_process():
    for unit in sorted(CSRC.glob("*.cu")):
        assert not re.search(r"static\s+(const\s+)?cudaError_t\s+\w+\s*=", unit.read_text()), unit.name


@pytest.mark.gpu
def test_operators_on_two_devices():
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    results = []
    for dev in ("cuda:0", "cuda:1"):
        gen = torch.Generator().manual_seed(1)
        x = torch.randn(40, 3, 4, 128, generator=gen).bfloat16().to(dev)
        table, lens = torch.arange(9, dtype=torch.int32, device=dev)[None], torch.tensor([40], dtype=torch.int32, device=dev)
        store, starts = PagedStore.allocate(40, 4, 16, 128, dev), torch.tensor([0, 40], dtype=torch.int32, device=dev)
        q = paged_append(store, x[:, 1], x[:, 2], table, lens, starts, q=x[:, 0])
        wide = table.expand(1, 9).repeat(1, 3)                      # a table of more than the keys that are not cut into pieces
        results.append([t.cpu() for t in (paged_attention(q, store, table, lens, starts), paged_attention(q[:1], store, wide, lens),
                                          sample(torch.randn(3, 50304, generator=gen).to(dev), torch.rand(3, generator=gen).to(dev), top_p=0.9))])
        _common.raise_on_device_error(torch.device(dev).index)
    assert all(torch.equal(a, b) for a, b in zip(*results))
