"""The host's side of paged attention, and what the kernels make of a call's arrays (csrc/paged.hpp), through the library
without a GPU: the work-groups and records that a call is given cover what its sequences ask for, whatever their lengths;
rows, positions and pages out of range stay out; scratch goes by the rows, sequences and heads alone."""
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "paged.hpp"
using namespace xtg::hip;
int main() {
  DevPaged c;
  PagedAttnCall a = {};
  int with_starts, cus;
  while (std::scanf("%d %d %d %d %d %d %d %d %d %d", &c.kv_heads, &c.pages, &c.shift, &a.heads, &a.seqs.n_seqs, &a.seqs.n_rows,
                    &a.seqs.max_pages, &a.window, &with_starts, &cus) == 10) {
    c.head_dim = 128, c.size = 1 << c.shift;
    std::vector<int> pos(a.seqs.n_seqs), starts(a.seqs.n_seqs + 1), table(size_t(a.seqs.n_seqs) * a.seqs.max_pages);
    for (int& x : pos) if (std::scanf("%d", &x) != 1) return 1;
    if (with_starts) for (int& x : starts) if (std::scanf("%d", &x) != 1) return 1;
    for (size_t x = 0; x < table.size(); ++x) table[x] = int(x * 7919 % 101) - 20;
    a.cache = &c, a.seqs.pos = pos.data(), a.seqs.starts = with_starts ? starts.data() : nullptr, a.seqs.table = table.data();
    a.seqs.pages = c.pages, a.seqs.shift = c.shift;
    const PagedPlan p = paged_plan(a, cus);
    PagedArgs k = {};
    k.s = a.seqs, k.group = a.heads / c.kv_heads, k.cols = p.cols, k.budget = p.budget, k.window = a.window;
    float total = 0;
    int blocks = 0;
    for (int s = 0; s < a.seqs.n_seqs; ++s) {
      const Extent x = extent(k, s);
      total += float(x.blocks) * float(x.tiles), blocks += x.blocks;
    }
    int chunk = first_chunk(k, total, blocks);
    for (int step = 0; step < kChunkSteps; ++step) {
      int n = 0;
      for (int s = 0; s < a.seqs.n_seqs; ++s) { const Extent x = extent(k, s); n += x.blocks * parts_of(x, chunk); }
      if (!next_chunk(k, chunk, n, blocks)) break;
    }
    long long tasks = 0, records = 0, bad = 0;
    for (int s = 0; s < a.seqs.n_seqs; ++s) {
      const Extent x = extent(k, s);
      const int n = parts_of(x, chunk);
      tasks += (long long)x.blocks * n;
      if (n > 1) records += (long long)x.blocks * n * x.cols(k);
      bad += (x.many && !p.many) || (!x.many && x.blocks > 1);
      bad += x.q.row0 < 0 || x.q.n < 0 || x.q.row0 + x.q.n > a.seqs.n_rows || x.tiles < 0 || x.lo < 0;
      bad += x.tiles > 0 && (x.lo + x.tiles) * 32 > a.seqs.max_pages << c.shift;
      for (int at : {0, x.q.pos, x.q.pos + x.q.n, kMostPositions - 1, (a.seqs.max_pages << c.shift) - 1, a.seqs.max_pages << c.shift}) {
        if (at < 0) continue;
        const int page = page_of(a.seqs, s, at);
        bad += page < -1 || page >= c.pages || (at >= a.seqs.max_pages << c.shift && page != -1);
      }
    }
    std::printf("%lld %d %lld %d %lld %zu\n", tasks, p.tasks, records, p.records, bad, p.bytes());
  }
}
"""


@pytest.fixture(scope="module")
def run(pkg, tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    "-I" + os.path.join(ROOT, "xtier-go_amd", "csrc"), str(d / "plan.cpp"), pkg.LIB_PATH,
                    "-Wl,-rpath," + os.path.dirname(pkg.LIB_PATH), "-L/opt/rocm/lib", "-lamdhip64", "-o",
                    str(d / "plan")], check=True)

    def go(calls):
        text = "".join("%d %d %d %d %d %d %d %d %d %d\n%s\n%s\n" % (
            *head, " ".join(map(str, pos)), " ".join(map(str, starts)) if head[8] else "") for head, pos, starts in calls)
        out = subprocess.run([str(d / "plan")], input=text, capture_output=True, text=True, check=True).stdout
        rows = [tuple(map(int, line.split())) for line in out.splitlines()]
        assert len(rows) == len(calls)
        return rows
    return go


def call(kvh, heads, pos, rows=None, window=0, max_pages=40, shift=6, cus=256, pages=60):
    starts = np.concatenate([[0], np.cumsum(rows)]) if rows is not None else []
    n_rows = int(starts[-1]) if rows is not None else len(pos)
    return (kvh, pages, shift, heads, len(pos), n_rows, max_pages, window, int(rows is not None), cus), list(pos), list(starts)


def test_tasks_and_records_cover_any_lengths(run):
    rng = np.random.default_rng(3)
    calls = []
    for _ in range(300):
        n, kvh = int(rng.integers(1, 300)), int(rng.choice([1, 2, 4, 8, 40]))
        heads, window = kvh * int(rng.choice([1, 2, 3, 4, 8, 17, 128])), int(rng.choice([0, 0, 1, 100, 1024]))
        top = int(rng.choice([1, 40, 2000, 40 * 64 + 500]))
        pos = rng.integers(-3, top, n)
        kind = rng.integers(0, 4)
        rows = None if kind == 0 else rng.integers(0, int(rng.choice([2, 9, 700])), n)
        if kind == 3:
            rows = np.zeros(n, np.int64)
            rows[rng.integers(0, n)] = 3000
        calls.append(call(kvh, heads, pos, rows, window, cus=int(rng.choice([1, 64, 256]))))
    for c, (tasks, most, records, room, bad, _) in zip(calls, run(calls)):
        assert tasks <= most and records <= room and bad == 0, (c, tasks, most, records, room, bad)


def test_arrays_out_of_range_stay_out(run):
    """Starts that decrease or pass the call's rows, positions near 2^31, tables with numbers that are no pages."""
    big = 2 ** 31 - 1
    calls = []
    for pos, starts in (([big, 5, -big - 1], [0, 2, 1, 9]), ([0, 0, 0], [-5, 100, big, -big]), ([big, big - 1, 2 ** 30], [0, 3, 6, 8]),
                        ([7, 7, 7], [8, 4, 2, 0])):
        head = (2, 60, 5, 8, 3, 8, 40, 0, 1, 256)
        for window in (0, 1, 50, big):
            calls.append((head[:7] + (window,) + head[8:], pos, starts))
    for c, (_, _, _, _, bad, _) in zip(calls, run(calls)):
        assert bad == 0, c


def test_scratch_goes_by_rows_sequences_and_heads(run):
    """A captured decode step's lengths change: the scratch of its first call is enough for all."""
    got = run([call(8, 32, [p] * 64, max_pages=4000) for p in (0, 31, 5000, 200000)] +
              [call(8, 32, [p] * 4, [512, 1, 1, 1], max_pages=4000) for p in (0, 31, 5000, 200000)])
    assert len({g[5] for g in got[:4]}) == 1 and len({g[5] for g in got[4:]}) == 1


def test_a_destroyed_pool_is_refused(pkg):
    """NULL handles are errors with a message, not calls (no GPU is asked)."""
    import ctypes
    lib, err = pkg.lib(), ctypes.create_string_buffer(200)
    rows, a, b = pkg.PagedRowsArgs(), pkg.PagedAppendArgs(), pkg.PagedAttnArgs()
    for rc in (lib.xtg_hip_paged_append(None, None, ctypes.byref(rows), ctypes.byref(a), err, 200),
               lib.xtg_hip_paged_read(None, None, ctypes.byref(rows), None, None, 0, err, 200),
               lib.xtg_hip_paged_attention(None, None, ctypes.byref(rows), ctypes.byref(b), err, 200),
               lib.xtg_hip_paged_globals(None, None, 1.0, 1.0, err, 200)):
        assert rc == -1 and b"NULL argument" in err.value
    assert not lib.xtg_hip_paged_create(None, 8, 128, 4, 64, 0, err, 200)
    lib.xtg_hip_paged_destroy(None, None)


class Ints:
    """An int32 array in the memory of device 0, for the checks of arguments alone."""
    dtype, shape = "torch.int32", ()

    def __init__(self, *shape):
        self.shape = shape

    def numel(self):
        return int(np.prod(self.shape))

    def is_contiguous(self):
        return True

    def get_device(self):
        return 0

    def data_ptr(self):
        return 4096


def test_starts_want_the_number_of_rows(pkg):
    """How many rows a call with starts has is in device memory: taken as one a sequence, those behind would be lost."""
    import types
    b = types.SimpleNamespace(device=0, h=1)
    assert pkg.PagedRows(b, Ints(3), Ints(3, 4)).n_rows == 3
    assert pkg.PagedRows(b, Ints(3), Ints(3, 4), 7, Ints(4)).n_rows == 7
    with pytest.raises(pkg.XtgError, match="n_rows"):
        pkg.PagedRows(b, Ints(3), Ints(3, 4), starts=Ints(4))


def test_arrays_of_a_closed_backend_are_refused(pkg):
    """Closing a backend frees its arrays, whose addresses stay: not to be read by another backend's calls."""
    import types
    made, other = types.SimpleNamespace(device=0, h=1), types.SimpleNamespace(device=0, h=1)

    def array(*shape):
        a = pkg.DeviceArray.__new__(pkg.DeviceArray)
        a.b, a.shape, a.dtype, a.ptr = made, shape, np.dtype(np.int32), 4096
        a.nbytes = 4 * int(np.prod(shape))
        return a
    rows = pkg.PagedRows(other, array(3), array(3, 4), 7, array(4))
    rows.of(other)
    made.h = None
    with pytest.raises(pkg.XtgError, match="have been freed"):
        rows.of(other)
    with pytest.raises(pkg.XtgError, match="pos has been freed"):
        pkg.PagedRows(other, array(3), array(3, 4), 7, array(4))


def test_rows_that_are_part_of_wider_ones(pkg, monkeypatch):
    """q, k and v as views of one projection's rows, with their stride; a stride that is not the view's, rows that are not
    packed, too few, of another type or on another device are refused. (Tensors of the CPU, whose device is -1, and a library
    that takes the call's arguments down.)"""
    import types
    torch = pytest.importorskip("torch")
    b = types.SimpleNamespace(device=-1, h=1, _err=None)
    got = []

    def taken(h, cache, rows, args, err, n):
        got.append(args._obj)
        return 0
    monkeypatch.setattr(pkg, "_lib", types.SimpleNamespace(xtg_hip_paged_append=taken, xtg_hip_paged_attention=taken))
    c = pkg.PagedCache.__new__(pkg.PagedCache)
    c.b, c.h, c.kv_heads, c.head_dim = b, 1, 2, 64
    rows = types.SimpleNamespace(n_rows=5, of=lambda backend: None)
    heads, width = 8, 12 * 64
    x = torch.zeros((6, width), dtype=torch.bfloat16)
    q, k, v = x[:, :512], x[:, 512:640], x[:, 640:]
    for shaped in (lambda y: y, lambda y: y.unflatten(1, (-1, 64))):
        c.append(rows, shaped(k), shaped(v), pkg.X_BF16, shaped(q), shaped(q), heads, 1e4, q_stride=width, k_stride=width, v_stride=width)
        c.attention(rows, shaped(q), torch.zeros((5, heads, 64), dtype=torch.bfloat16), heads, pkg.X_BF16, q_stride=width)
        for a in got:
            assert a.q == x.data_ptr() and a.q_stride == width
        assert (got[0].k, got[0].v, got[0].q_out) == (x.data_ptr() + 1024, x.data_ptr() + 1280, x.data_ptr())
        del got[:]
    c.append(rows, x[:5], v, pkg.X_BF16, k_stride=width, v_stride=width)   # the whole rows' first elements

    def refused(match, k, v=v, stride=width, x_dtype=pkg.X_BF16):
        with pytest.raises(pkg.XtgError, match=match):
            c.append(rows, k, v, x_dtype, k_stride=stride, v_stride=width)
    refused("768 elements apart, not the call's 776", k, stride=776)
    refused("k has 4 rows, the call 5", k[:4])
    refused("64 elements, the call's rows of it take 128", k[:, :64])
    refused("not contiguous", x[:, 512::2])
    refused("not contiguous", x[:5].T)
    refused("not of the call's row type BF16", x.float()[:, 512:640])
    with pytest.raises(pkg.XtgError, match="not contiguous"):
        c.append(rows, k, v, pkg.X_BF16)
    b.device = 0
    refused("not in the memory", k)


@pytest.fixture(scope="module")
def run_of(pkg, tmp_path_factory):
    """The program for heads of other sizes, as functions of calls (their texts' lines to the program's numbers)."""
    def made(d):
        at = tmp_path_factory.mktemp("paged%d" % d)
        (at / "plan.cpp").write_text(PROGRAM.replace("c.head_dim = 128", "c.head_dim = %d" % d))
        csrc = os.path.join(ROOT, "xtier-go_amd", "csrc")
        subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + csrc, str(at / "plan.cpp"),
                        pkg.LIB_PATH, "-Wl,-rpath," + os.path.dirname(pkg.LIB_PATH), "-L/opt/rocm/lib", "-lamdhip64", "-o",
                        str(at / "plan")], check=True)

        def go(calls):
            text = "\n".join(" ".join(map(str, [*head, *pos, *(starts if head[8] else [])])) for head, pos, starts in calls)
            out = subprocess.run([str(at / "plan")], input=text, capture_output=True, text=True, check=True).stdout
            return [tuple(map(int, line.split())) for line in out.splitlines()]
        return go
    return {d: made(d) for d in (64, 256)}


def test_scratch_goes_by_what_the_header_names(run, run_of):
    """A call alike in rows, sequences, heads, starts (NULL or not), the pool's KV heads and dims and tables for more than 128
    positions needs as much as the first such call, whatever the pages' size and number, the tables' length, the window and
    the positions."""
    rng = np.random.default_rng(4)
    alike = [(kvh, kvh * group, n, rows) for kvh in (1, 8) for group in (1, 4, 40)
             for n, rows in ((1, None), (70, None), (70, np.ones(70, int)), (3, np.array([300, 1, 0])), (9, np.array([8] * 9)))]
    for go in (run, run_of[64], run_of[256]):
        calls = [call(kvh, heads, rng.integers(0, 5000, n), rows, window=w, max_pages=m, shift=s, pages=p)
                 for kvh, heads, n, rows in alike for w, m, s, p in ((0, 40, 6, 60), (100, 3, 12, 7), (1024, 5, 5, 1000))]
        got = [r[5] for r in go(calls)]
        assert len(got) == len(calls) and all(len(set(got[i:i + 3])) == 1 for i in range(0, len(got), 3))


def test_tasks_and_records_cover_any_lengths_of_other_heads(run_of):
    """As for heads of 128 dims; those of 256 go in blocks of 16 q-cols beside blocks of many."""
    rng = np.random.default_rng(5)
    for go in run_of.values():
        calls = []
        for _ in range(200):
            n, kvh = int(rng.integers(1, 200)), int(rng.choice([1, 2, 4, 8]))
            heads, window = kvh * int(rng.choice([1, 2, 3, 8, 17, 24, 32, 128])), int(rng.choice([0, 0, 100, 1024]))
            rows = [None, rng.integers(0, 2, n), rng.integers(2, 17, n), rng.integers(0, 500, n)][int(rng.integers(0, 4))]
            calls.append(call(kvh, heads, rng.integers(-3, 2500, n), rows, window, cus=int(rng.choice([1, 64, 256]))))
        for c, (tasks, most, records, room, bad, _) in zip(calls, go(calls)):
            assert tasks <= most and records <= room and bad == 0, (c, tasks, most, records, room, bad)


def test_a_chunk_beside_single_tokens_is_cut(run, run_of):
    """The calls that the GPU's test of the merges makes have records: their chunks' blocks are in several parts."""
    for go in (run, run_of[64], run_of[256]):
        for rows, ctx in ((260, 4000), (40, 4000)):
            calls = [call(4, 32, [ctx, 900, 30, 2000], [rows, 1, 1, 1], max_pages=70), call(4, 32, [ctx], [rows], max_pages=70)]
            blocks = -(-rows * 8 // 128)
            for (tasks, _, records, room, bad, _) in go(calls):
                assert tasks >= 2 * blocks and room >= records >= 2 * blocks * 128 and bad == 0
