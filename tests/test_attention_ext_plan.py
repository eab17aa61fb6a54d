"""The host-side plan of an attention call with changed scores (ext_plan in csrc/attention_ext.hip), through the library
without a GPU: the scratch it asks for covers what the call writes and is the same at every position of a cache, with or
without a window (a decode loop, or a graph captured after an early call, must not outgrow it)."""
import collections
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include "attention_ext.hpp"
int main() {
  xtg::hip::DevKv c;
  xtg::hip::ExtCall a = {};
  int ring, own, end, cus;
  while (std::scanf("%d %d %lld %d %d %d %lld %d %d %d %d", &c.kv_heads, &c.head_dim, &c.slots, &ring, &a.n_q, &a.heads,
                    &a.pos0, &a.window, &own, &end, &cus) == 11) {
    c.ring = ring, c.slots_pad = int((c.slots + 31) / 32 * 32);
    a.cache = c.slots ? &c : nullptr, a.kv_heads = c.kv_heads, a.d = c.head_dim;
    a.k = a.v = own ? &c : nullptr, a.end = end ? &ring : nullptr;
    const xtg::hip::ExtPlan p = xtg::hip::ext_plan(a, cus);
    std::printf("%d %d %d %d %zu %zu\n", int(p.few), p.tiles, p.splits, p.own, p.used_bytes(), p.scratch);
  }
}
"""
Plan = collections.namedtuple("Plan", "few tiles splits own used scratch")


@pytest.fixture(scope="module")
def plans(pkg, tmp_path_factory):
    """plans([(kv_heads, head_dim, slots (0: no cache), ring, n_q, heads, pos0, window, own keys, end given, CUs)])"""
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    "-I" + os.path.join(ROOT, "xtier-go_amd", "csrc"), str(d / "plan.cpp"), pkg.LIB_PATH,
                    "-Wl,-rpath," + os.path.dirname(pkg.LIB_PATH), "-L/opt/rocm/lib", "-lamdhip64", "-o",
                    str(d / "plan")], check=True)

    def run(calls):
        text = "\n".join(" ".join(str(int(v)) for v in c) for c in calls) + "\n"
        r = subprocess.run([str(d / "plan")], input=text, capture_output=True, text=True, check=True)
        out = [Plan(*map(int, line.split())) for line in r.stdout.splitlines()]
        assert len(out) == len(calls)
        return out

    return run


@pytest.mark.parametrize("heads,kv,d", [(32, 8, 128), (16, 4, 256), (16, 8, 64), (8, 8, 128), (2, 1, 128), (32, 1, 64), (64, 8, 256)])
@pytest.mark.parametrize("slots,ring", [(1040, 1), (700, 1), (9000, 0), (40000, 0)])
def test_scratch_is_the_same_at_every_position(plans, heads, kv, d, slots, ring):
    for n_q in (1, 3, 5, 8, 20, 45, 188, 512):
        last = 3 * slots if ring else slots - n_q
        at = [p for p in {0, 1, 31, 33, 128, 512, 1000, 1039, 1041, 5000, slots // 2, slots - 1, slots + 1, last} if 0 <= p <= last]
        for own in (0, 1):
            calls = [(kv, d, slots, ring, n_q, heads, pos, w, own, end, 256) for pos in at for w in (0, 300, 4096) for end in (0, 1)]
            ps = plans(calls)
            assert len({p.scratch for p in ps}) == 1, (n_q, own, sorted(zip(calls, ps))[:3])
            assert all(p.used <= p.scratch for p in ps)
            assert ps[0].scratch < 128 << 20


def test_a_call_of_its_own_keys_needs_what_it_writes(plans):
    for n_q in (1, 40, 300, 2000):
        for p in plans([(8, 128, 0, 0, n_q, 32, pos, w, 1, 0, 256) for pos in (0, 1000) for w in (0, 50)]):
            assert p.used == p.scratch and p.splits <= 4
