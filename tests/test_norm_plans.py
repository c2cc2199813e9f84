"""Host-side decisions of the group-norm and dropout kernels, called as they are from a small program: no GPU needed."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "l_inf-dist-net_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include "group_norm.cuh"
namespace linf { int sm_count() { return 148; } std::atomic<unsigned long long> g_launches{0}; }
using namespace linf;
int main(int argc, char** argv) {
    if (!strcmp(argv[1], "drop")) {                 // rate, whether a state is given -> on, which pointer
        static const long long idle[2] = {0, 0}, rng[2] = {1, 2};
        Drop d;
        if (!make_drop(atof(argv[2]), atoi(argv[3]) ? rng : nullptr, idle, &d)) return printf("refused"), 0;
        printf("%d %s", d.on, d.rng == rng ? "rng" : d.rng == idle ? "idle" : "null");
    }
    if (!strcmp(argv[1], "params")) printf("%u", norm_param_ctas(atoi(argv[2])));
    return 0;
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    """ask("what", ...) -> what the program prints."""
    at = tmp_path_factory.mktemp("plans")
    source, program = at / "plans.cu", at / "plans"
    source.write_text(PROGRAM)
    subprocess.check_call(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", CSRC, "-o", str(program), str(source)])

    def call(*words):
        return subprocess.run([str(program), *map(str, words)], capture_output=True, text=True, timeout=20, check=True).stdout.split()
    return call


@pytest.mark.parametrize("rate, given, want", [(0.0, 0, ["0", "idle"]), (0.0, 1, ["0", "idle"]), (2.0 ** -18, 1, ["0", "idle"]),
                                               (0.5, 1, ["1", "rng"]), (1.0, 1, ["1", "rng"]), (1.5, 1, ["refused"])])
def test_no_kernel_holds_a_null_generator_state(ask, rate, given, want):
    """Where nothing is dropped a valid address stands for the state, so that a load moved in front of its condition reads nothing it must not."""
    assert ask("drop", rate, given) == want


@pytest.mark.parametrize("channels", [1, 8, 9, 2 ** 31 - 8, 2 ** 31 - 7, 2 ** 31 - 1])
def test_ctas_of_the_parameters_gradients(ask, channels):
    """All channel counts that a call may have, the last seven below 2^31 among them."""
    assert ask("params", channels) == [str(-(-channels // 8))]


@pytest.mark.parametrize("call", ["group_norm_workspace_bytes(1, 2**30 + 1, 1, 1, 0, 0)", "group_norm_workspace_bytes(1, 2**31 - 1, 1, 1, 1, 1)",
                                  "group_norm_workspace_bytes(1, 2**31 - 2, 1, 1, 2, 1)", "group_norm_bound_workspace_bytes(1, 2**31 - 1, 1, 1, 1)"])
def test_rows_of_a_thousand_million_channels_are_planned(lib, call):
    """In a process of its own, which ends in time."""
    code = f"import linfdist_b200 as L; assert L._lib.load().linf_{call} >= 0"
    subprocess.run(["python", "-c", code], cwd=os.path.dirname(os.path.dirname(CSRC)), timeout=60, check=True)
