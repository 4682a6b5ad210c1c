"""Work that a launcher does once per device (lt_once.cuh), compiled for the host with devices of its own."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))

PROGRAM = r"""
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>
#include "lt_once.cuh"
static thread_local int device = 0;
extern "C" cudaError_t cudaGetDevice(int* d) { *d = device; return device < 0 ? cudaErrorNoDevice : cudaSuccess; }
static std::atomic<int> begun{0}, ended{0}, early{0};
static lt::PerDeviceOnce once;
static int launcher(int dev) {
    device = dev;
    LT_ONCE(once, begun++; std::this_thread::sleep_for(std::chrono::milliseconds(100)); ended++);
    if (ended == 0) early++;         // would launch ahead of the work
    return 0;
}
static int failing = 1;
static lt::PerDeviceOnce again;
static int refused(int dev) {
    device = dev;
    LT_ONCE(again, if (failing) return 7);
    return 0;
}
int main() {
    std::vector<std::thread> t;
    for (int i = 0; i < 8; i++) t.emplace_back(launcher, 3);
    for (auto& x : t) x.join();
    std::printf("%d %d %d\n", (int)begun, (int)ended, (int)early);      // eight threads, one device
    launcher(3); launcher(4); launcher(4);
    std::printf("%d\n", (int)begun);                                    // another device
    launcher(64); launcher(64); launcher(-1);
    std::printf("%d\n", (int)begun);                                    // devices that are not remembered
    std::printf("%d %d", refused(0), refused(0));                       // work that fails is not done
    failing = 0;
    std::printf(" %d", refused(0));
    failing = 1;
    std::printf(" %d %d\n", refused(0), refused(1));
}
"""


def test_every_launch_waits_for_the_work(tmp_path):
    src, exe = tmp_path / "once.cpp", str(tmp_path / "once")
    src.write_text(PROGRAM)
    include = [a for d in ("/usr/local/cuda/include", os.path.join(HERE, "..", "llamatov_b200", "csrc")) for a in ("-I", d)]
    subprocess.run(["g++", "-std=c++17", "-pthread", *include, str(src), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, check=True, timeout=60).stdout.split("\n")[:4]
    assert out == ["1 1 0", "2", "5", "7 7 0 0 7"]
