"""What the operators over decisions hold and launch, without a GPU: on a HIP runtime in host
memory, whose kernels do nothing."""
import json
import os
import subprocess
import sys
import textwrap

import pytest
from test_host_memory import HERE, PRELUDE, host  # noqa: F401  (fixture)
from test_policy_refusals import SETUP

CALLS = """
    MB = 1 << 20
    fake.fake_live_bytes.restype = c_uint64
    def prefer(n, classes=10):
        ok(lib.dp_preference_loss(ws, rows(n_rows=n, n_classes=classes, row_stride=classes), P,
                                  c_int64(2), None, byref(Preference(0.1, 0.0, 0)), P, None, None,
                                  P, None, None))
    def split(channels):
        r = Recurrence(1, 100000, channels, 0, 0)
        for i in range(5):
            r.strides[i][0], r.strides[i][1] = 100000 * channels, channels
        ok(lib.dp_linear_recurrence(ws, byref(r), P, P, None, P, None, None))
    def long_rows(n, classes):
        ok(lib.dp_action_logprobs(ws, rows(n_rows=n, n_classes=classes, row_stride=classes), P,
                                  None, None))
    live = lambda: fake.fake_live_bytes(0)
"""


@pytest.mark.parametrize("first", ["prefer(1000)", "split(8)", "long_rows(4, 40000)"])
def test_scratch_of_captured_calls_lives_as_long_as_the_workspace(host, first):  # noqa: F811
    """A graph uses the block that it was captured with: what outgrows it must not free it."""
    got = host(SETUP + CALLS + f"""
    start = live()
    {first}
    small = live()
    prefer(200000)
    prefer(100)
    grown = live()
    prefer(400000)
    prefer(400000)
    most = live()
    ok(lib.dp_workspace_free(ws))
    print(json.dumps([start, small, grown, most, live()]))
    """)
    mb = 1 << 20
    start, small, grown, most, end = (x - got[0] for x in got)
    assert small == mb and grown == mb + 4 * mb and most == mb + 4 * mb + 8 * mb and end == 0


def test_scratch_of_other_calls_is_replaced(host):  # noqa: F811
    """Calls that cannot be captured leave nothing behind when they outgrow their scratch."""
    got = host(SETUP + CALLS + """
    param = (c_double * 8)()
    start = live()
    seen = []
    for nodes in (100, 400, 1600):  # 32 bytes a feature of a node
        ok(lib.dp_evaluate_splits(ws, P, nodes, 500, 256, P, P, 0, 0, byref(param), P, None))
        seen.append((live() - start) // MB)
    prefer(1000)
    ok(lib.dp_evaluate_splits(ws, P, 3200, 500, 256, P, P, 0, 0, byref(param), P, None))
    print(json.dumps(seen + [(live() - start) // MB]))
    """)
    assert got == [2, 8, 32, 32 + 64]


def test_a_growth_that_finds_no_memory_leaves_the_scratch(host):  # noqa: F811
    got = host(SETUP + CALLS + """
    prefer(1000)
    before = live()
    fake.fake_fail_after(0)
    failed = lib.dp_preference_loss(ws, rows(n_rows=200000), P, c_int64(2), None,
                                    byref(Preference(0.1, 0.0, 0)), P, None, None, P, None, None)
    prefer(1000)  # needs no memory
    fake.fake_fail_after(-1)
    print(json.dumps([failed, live() - before]))
    """)
    assert got[0] != 0 and got[1] == 0


# Allocations of the runtime in host memory take address space only: the scratch of very many
# rows, which no kernel touches there.
RESERVE = """
#include <cstdlib>
#include <sys/mman.h>
namespace std {
inline void* reserve(size_t count, size_t bytes) {
  void* p = mmap(nullptr, count * bytes, PROT_READ | PROT_WRITE,
                 MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
  return p == MAP_FAILED ? nullptr : p;
}
}
#define calloc reserve
"""


@pytest.fixture(scope="session")
def vast(dp, tmp_path_factory):
    """Runs code as `host` does, with allocations of any size."""
    folder = tmp_path_factory.mktemp("vast")
    header, fake = folder / "reserve.hpp", folder / "libfake_hip.so"
    header.write_text(RESERVE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", "-include", str(header), "-o", str(fake),
                    os.path.join(HERE, "native", "fake_hip.cpp")], check=True)

    def run(code):
        text = PRELUDE.format(fake=str(fake), lib=dp.LIB_PATH) + textwrap.dedent(code)
        p = subprocess.run([sys.executable, "-c", text], capture_output=True, text=True,
                           timeout=120)
        assert p.returncode == 0, p.stderr
        return json.loads(p.stdout)

    return run


@pytest.mark.parametrize("pairs,rows,lanes", [(2 ** 31 - 1, 0, 1), (2 ** 31 - 1, 3, 2),
                                              (1 << 30, 5, 4), (1 << 26, 65, 64), (5000, 3, 2)])
def test_pairs_are_launched_in_parts_that_a_grid_holds(vast, pairs, rows, lanes):
    """A launch has fewer than 2^32 threads, also where each of very many pairs takes several."""
    got = vast(SETUP + f"""
    ok(lib.dp_preference_loss(ws, rows(n_rows={pairs * rows}, n_classes=1, row_stride=1, dtype=1),
                              P, c_int64({pairs}), None, byref(Preference(0.1, 0.0, 0)), P, None,
                              None, P, None, None))
    seen = [x.split(" ") for x in fake.fake_launches().decode().split(";") if x]
    print(json.dumps([[n, int(g.split(",")[0]), int(b)] for n, g, b in seen]))
    """)
    assert all(grid * block < 2 ** 32 for _, grid, block in got)
    threads = sum(grid * block for name, grid, block in got if "pair_kernel" in name)
    assert 0 <= threads - lanes * pairs < 256
