"""The 8-bit linear layer's ring of stages: no barrier's arrival is left on its way when a CTA leaves.

The tensor core releases a stage by an arrival of its own, which nothing orders before the accumulator's.
The producer's walk over the ring (csrc/ring.cuh, compiled here by the host's compiler) is run against
modelled barriers whose arrivals come as late as a wait allows.
"""
import os
import re
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "streaming_sparse_b200", "csrc")

MODEL = r"""
#include "ring.cuh"

#include <cstdio>
#include <vector>

struct Barrier {   // one arrival a phase; a wait for a parity ends once the phase of that parity is complete
    int sent = 0, landed = 0;
    bool wait(uint32_t parity) {
        while ((uint32_t)(landed & 1) == parity) {   // the phase under way has it: arrivals land until it is complete
            if (landed == sent) return false;        // never: nothing that could land is on its way
            ++landed;
        }
        return true;
    }
};

int main() {
    for (int n = 1; n <= 10; ++n)
        for (int steps = 0; steps <= 4 * n + 1; ++steps) {
            std::vector<Barrier> released(n);
            ss::Ring ring{n};
            int issued = 0;
            for (int k = 0; k < steps; ++k) {
                if (k >= n && !released[ring.at].wait(ring.parity ^ 1u)) return std::printf("stuck %d %d\n", n, steps);
                ++released[ring.at].sent;   // the load, and in its time the release of the stage by its product
                ring.next();
                issued = issued + 1 < n ? issued + 1 : n;
            }
            std::vector<int> seen;
            if (!ring.wait_for_each(issued, [&](int at, uint32_t parity) {
                    seen.push_back(at);
                    return released[at].wait(parity);
                }))
                return std::printf("a wait without an arrival: %d stages, %d steps\n", n, steps);
            for (auto &b : released)
                if (b.landed != b.sent) return std::printf("left on its way: %d stages, %d steps\n", n, steps);
            if ((int)seen.size() != issued) return std::printf("%d of %d\n", (int)seen.size(), issued);
            if (issued && !ring.wait_for_each(issued, [&](int, uint32_t) { return true; })) return 1;
            int calls = 0;
            if (issued && ring.wait_for_each(issued, [&](int, uint32_t) { ++calls; return false; })) return 2;
            if (calls != (issued ? 1 : 0)) return std::printf("went on after a wait that ran out\n");
        }
    std::printf("ok");
    return 0;
}
"""


def test_the_walk_waits_for_every_release(tmp_path):
    src, exe = tmp_path / "model.cpp", tmp_path / "model"
    src.write_text(MODEL)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert (r.returncode, r.stdout) == (0, "ok"), r.stdout


def test_every_producer_takes_the_walk_before_it_leaves():
    """Both kernels' producers wait for the releases (EMPTY) where nothing went wrong, not only after a timeout."""
    with open(os.path.join(CSRC, "linear_i8.cu")) as f:
        code = f.read()
    producers = re.findall(r"ring\.next\(\);\s*issued = min\(issued \+ 1, nst\);(.*?)report\(p\.status", code, re.S)
    assert len(producers) == 2
    for rest in producers:
        assert re.search(r"if \(ok\)\s*ok = ring\.wait_for_each\(issued,.*?EMPTY \+ at", rest, re.S)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 40, 130, 700, 2600])
def test_sums_at_every_fill_of_the_ring(M):
    """One step to more than twice the ring's stages, several tiles a pair: no wait runs out and every sum is exact."""
    from streaming_sparse_b200 import ops

    dev, N = torch.device("cuda:0"), 1100
    g = torch.Generator(device=dev).manual_seed(M)
    for steps in (1, 2, 3, 4, 5, 6, 7, 9, 10, 11, 12, 13, 19, 20, 21, 23):
        K = 128 * steps - (steps % 3) * 16
        x = torch.randint(-127, 128, (M, K), device=dev, generator=g).to(torch.int8)
        w = torch.randint(-127, 128, (N, K), device=dev, generator=g).to(torch.int8)
        one = torch.ones(max(M, N), device=dev)
        got = ops.linear_i8(x, one[:M], w, one[:N], out_dtype=torch.float32, validate=True)
        assert torch.equal(got, (x.double() @ w.double().t()).float())
