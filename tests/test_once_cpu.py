"""CPU: the once-per-device action of the launchers (nncf_amd/csrc/wc_once.h), compiled for the host: a second thread waits for the
first one's action, a failed action is tried again."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nncf_amd", "csrc")
PROGRAM = r"""
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>
#include "wc_once.h"
int main() {
    int bad = 0;
    for (int round = 0; round < 20; ++round) {
        wc::OncePerKey once;
        std::atomic<int> runs{0}, finished{0}, early{0};
        std::vector<std::thread> threads;
        for (int t = 0; t < 8; ++t)
            threads.emplace_back([&] {
                const bool ok = once.run(3, [&] {
                    ++runs;
                    std::this_thread::sleep_for(std::chrono::milliseconds(5));
                    ++finished;
                    return true;
                });
                if (!ok || finished.load() != 1) ++early;
            });
        for (auto& t : threads) t.join();
        bad += early.load() + (runs.load() != 1);
    }
    wc::OncePerKey once;
    int calls = 0;
    bad += once.run(0, [&] { ++calls; return false; }) ? 1 : 0;
    bad += once.run(0, [&] { ++calls; return true; }) ? 0 : 1;
    bad += once.run(0, [&] { ++calls; return false; }) ? 0 : 1;  // done: not asked again
    bad += once.run(1, [&] { ++calls; return true; }) ? 0 : 1;   // another device
    for (int key : {-1, 64}) for (int i = 0; i < 2; ++i) once.run(key, [&] { ++calls; return true; });
    bad += calls != 7;
    std::printf("%d\n", bad);
    return 0;
}
"""


def test_the_second_thread_waits_for_the_first(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    (tmp_path / "once.cpp").write_text(PROGRAM)
    subprocess.check_call([gxx, "-std=c++17", "-O1", "-pthread", "-I", CSRC, str(tmp_path / "once.cpp"), "-o", str(tmp_path / "once")])
    assert subprocess.check_output([str(tmp_path / "once")], timeout=60).decode().strip() == "0"


def test_every_launcher_uses_it():
    """No launcher asks for the attribute outside of such an action."""
    for name in sorted(os.listdir(CSRC)):
        if name.endswith(".hip"):
            text = open(os.path.join(CSRC, name)).read()
            assert "first_on_device" not in text, name
            if "hipFuncSetAttribute(" in text:
                assert "once" in text and ".run([&]" in text, name
