"""The group norm's division of work (csrc/group_norm_plan.h, compiled for the host): for every size the blocks
tile the channels, the packs lie within rows and blocks, a block's threads cover it, and the rows that a workgroup
holds or the runs of positions cover the sample."""

import subprocess
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "myflows_amd" / "csrc"

PROBE = r"""
#include <cstdio>
#include "group_norm_plan.h"
using namespace mfh;

const char* fault(const GroupNormShape& s, int size, bool backward) {
    const GroupNormPlan p = group_norm_plan(s, size, backward);
    const int lanes = p.lanes, step = lanes > 0 ? p.threads / lanes : 0;
    if (p.vw < 1 || p.vw * size > 16 || s.channels % p.vw || p.width % p.vw) return "pack";
    if (lanes <= 32 && (lanes & (lanes - 1))) return "lanes that join across a wave";
    if (lanes > p.threads || lanes * p.vw < p.width || step < 1) return "lanes";
    if (p.groups < 1 || p.groups > p.threads || p.groups > GROUP_NORM_BLOCK_GROUPS) return "groups";
    if (p.parts == 1) {
        if (p.width != p.groups * p.per || static_cast<long long>(p.blocks) * p.width != s.channels) return "blocks";
    } else if (p.held || p.groups != 1 || p.blocks != s.groups * p.parts || p.per % p.vw ||
               static_cast<long long>(p.parts - 1) * p.width >= p.per || static_cast<long long>(p.parts) * p.width < p.per) {
        return "parts";
    }
    if (p.held) {
        if (static_cast<long long>(step) * group_norm_hold(size, p.vw, backward, p.threads) < s.positions) return "held rows";
    } else {
        if (p.threads != GROUP_NORM_SPLIT_THREADS || p.rows < 1 || p.runs < 1) return "runs";
        if (static_cast<long long>(p.runs) * p.rows < s.positions || static_cast<long long>(p.runs - 1) * p.rows >= s.positions)
            return "run rows";
    }
    return nullptr;
}

int main() {
    const int pers[] = {1, 2, 3, 5, 7, 8, 15, 16, 31, 33, 64, 65, 100, 127, 128, 255, 256, 257, 511, 512, 999, 1000, 1023,
                        1024, 1025, 2047, 2048, 2049, 4095, 4096, 5000, 8192, 16384, 40000, 65535, 65536};
    const int groups[] = {1, 2, 3, 4, 5, 6, 8, 11, 13, 16, 32, 64, 100, 256, 257, 512, 1024, 4096, 65536};
    const int positions[] = {1, 2, 3, 8, 20, 64, 100, 405, 1131, 4096, 16384, 100000, 1000000, 2147483647};
    long plans = 0, held = 0;
    for (int size : {2, 4})
        for (bool backward : {false, true})
            for (long long n : {1LL, 2LL, 7LL, 64LL, 300LL, 5000LL, 100000LL, 16777216LL})
                for (int per : pers)
                    for (int g : groups)
                        for (int at : positions) {
                            const long long channels = static_cast<long long>(per) * g;
                            if (channels > 65536 || channels * at > 2147483647LL || n * channels > (1LL << 28)) continue;
                            const GroupNormShape s{n, at, static_cast<int>(channels), g};
                            ++plans;
                            held += group_norm_plan(s, size, backward).held;
                            if (const char* what = fault(s, size, backward)) {
                                std::printf("%s: n %lld positions %d channels %lld groups %d size %d backward %d\n", what, n, at,
                                            channels, g, size, backward);
                                return 1;
                            }
                        }
    std::printf("%ld %ld\n", plans, held);
    return 0;
}
"""


def test_every_plan_covers_its_sample(tmp_path):
    source = tmp_path / "probe.cpp"
    source.write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", str(CSRC), str(source), "-o", str(tmp_path / "probe")], check=True)
    result = subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, timeout=100)
    assert result.returncode == 0, result.stdout
    plans, held = map(int, result.stdout.split())
    assert 0 < held < plans


LIMITS = r"""
#include <cstdio>
#include "group_norm_plan.h"
using namespace mfh;

int main() {
    const int pers[] = {1, 2, 3, 8, 15, 64, 255, 1000, 2048, 4096, 8192, 8193, 16384, 40000, 65535, 65536};
    const int groups[] = {1, 2, 3, 8, 32, 256, 257, 1024, 8192, 65536};
    const int positions[] = {1, 2, 20, 405, 4096, 40000, 1000000, 1073741824};
    const long long samples[] = {1, 7, 300, 2049, 4096, 20000, 65536, 1048576, 16777216, 16777224, 268435456};
    const long long most = 4294967295LL;  // threads of a launch
    long sliced = 0;
    for (int size : {2, 4})
        for (bool backward : {false, true})
            for (long long n : samples)
                for (int per : pers)
                    for (int g : groups)
                        for (int at : positions) {
                            const long long channels = static_cast<long long>(per) * g;
                            if (channels > 65536 || channels * at > 2147483647LL || n * channels > (1LL << 28)) continue;
                            const GroupNormShape s{n, at, static_cast<int>(channels), g};
                            const GroupNormPlan p = group_norm_plan(s, size, backward);
                            const long long slice = group_norm_slice(s, p, backward), count = slice < n ? slice : n;
                            // Every launch of a call, as csrc/group_norm.hip issues them.
                            const long long pass = count * p.blocks * (p.held ? 1 : p.runs) * p.threads;
                            const long long stats = p.held || backward ? 0 : count * g * 256;
                            const long long columns = p.held || !backward ? 0 : count * ((2 * channels + 63) / 64) * 1024;
                            sliced += slice < n;
                            if (slice >= 1 && pass <= most && stats <= most && columns <= most) continue;
                            std::printf("n %lld positions %d channels %lld groups %d size %d backward %d: slices of %lld, %lld "
                                        "%lld %lld threads\n", n, at, channels, g, size, backward, slice, pass, stats, columns);
                            return 1;
                        }
    std::printf("%ld\n", sliced);
    return 0;
}
"""


def test_every_launch_of_every_accepted_size_is_one_that_can_be_issued(tmp_path):
    source = tmp_path / "limits.cpp"
    source.write_text(LIMITS)
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", str(CSRC), str(source), "-o", str(tmp_path / "limits")], check=True)
    result = subprocess.run([str(tmp_path / "limits")], capture_output=True, text=True, timeout=100)
    assert result.returncode == 0, result.stdout
    assert int(result.stdout) > 0  # sizes beyond one launch are among them
