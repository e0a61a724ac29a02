"""CPU: how the paged attention kernels share a line of units among workers.
The device code's own arithmetic (csrc/share.cuh), compiled for the host,
against whole numbers of any size."""

import random
import shutil
import subprocess

import pytest

from conftest import PKG

MAIN = r"""
#include <inttypes.h>
#include <stdio.h>
#include "share.cuh"
int main() {
  char f;
  int64_t a, b, c;
  while (scanf(" %c %" SCNd64 " %" SCNd64 " %" SCNd64, &f, &a, &b, &c) == 4)
    printf("%" PRId64 "\n", f == 'm' ? q6w::paged::muldiv(a, b, c) : q6w::paged::owner_of(a, b, c));
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("shares")
    (d / "main.cpp").write_text(MAIN)
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no host compiler")
    subprocess.run([gxx, "-std=c++17", "-I", str(PKG / "csrc"), str(d / "main.cpp"), "-o", str(d / "main")], check=True)

    def run(calls):
        text = "\n".join(" ".join(map(str, c)) for c in calls)
        out = subprocess.run([str(d / "main")], input=text, capture_output=True, text=True, check=True).stdout
        return [int(x) for x in out.split()]

    return run


def numbers(rng, most):
    return rng.choice([rng.randrange(1, most), int(2 ** rng.uniform(0, most.bit_length() - 1)), most - 1, 1])


def test_muldiv(host):
    rng = random.Random(1)
    calls = [("m", 30 * 33404851, 1, 4943917969),  # a product of 32 bits, a divisor of 33
             ("m", 0, 1, 1 << 32), ("m", 5, 1, (1 << 32) + 1), ("m", (1 << 32) - 1, 1, 1 << 32),
             ("m", 1 << 32, 1, 1 << 32), ("m", (1 << 32) - 1, 1, (1 << 32) - 1), ("m", 147, 4943917969, 148)]
    calls += [("m", numbers(rng, 1 << 34), numbers(rng, 1 << 11), numbers(rng, 1 << 36)) for _ in range(4000)]
    assert host(calls) == [a * b // c for _, a, b, c in calls]


def test_owner_of(host):
    """The worker whose stretch [w units / workers, (w + 1) units / workers) holds a unit."""
    rng = random.Random(2)
    calls = []
    for _ in range(4000):
        units = numbers(rng, 1 << 36)
        workers = min(rng.choice([1, 147, 148, 2368]), units)
        w = rng.randrange(workers)
        first, end = w * units // workers, (w + 1) * units // workers
        calls += [("o", u, units, workers) for u in {first, end - 1, rng.randrange(first, end)}]
    got = host(calls)
    for (_, u, units, workers), w in zip(calls, got):
        assert w * units // workers <= u < (w + 1) * units // workers
