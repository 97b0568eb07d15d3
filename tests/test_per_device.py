"""Settings that HIP keeps for each device (the LDS a kernel may use) are made on each device that launches (p8x_once.h). CPU only:
a C++ program built with g++ and a look at the sources."""
import glob
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pingala8-llm_amd", "csrc")


def test_once_on_each_device(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(r"""
#include <atomic>
#include <cassert>
#include <cstdio>
#include <thread>
#include "p8x_once.h"
int main() {
    p8x::OncePerDevice o;
    int calls = 0;
    auto ok = [&] { ++calls; return 0; };
    auto bad = [&] { ++calls; return -3; };
    assert(o.run(0, ok) == 0 && calls == 1);
    assert(o.run(0, ok) == 0 && calls == 1);      // made already
    assert(o.run(2, ok) == 0 && calls == 2);      // another device: made there too
    assert(o.run(1, bad) == -3 && calls == 3);    // an error is reported and not kept
    assert(o.run(1, ok) == 0 && calls == 4);
    assert(o.run(1, bad) == 0 && o.run(0, bad) == 0 && o.run(2, bad) == 0 && calls == 4);
    p8x::OncePerDevice t;                         // callers on several threads: one of them makes it, none returns before that
    std::atomic<int> made{0}, n{0};
    std::thread th[8];
    for (auto &x : th) x = std::thread([&] { for (int d = 0; d < 4; ++d) { assert(t.run(d, [&] { ++n; ++made; return 0; }) == 0); assert(made > d); } });
    for (auto &x : th) x.join();
    assert(n == 4);
    puts("ok");
}
""")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-pthread", "-I", CSRC, str(src), "-o", str(exe)], check=True, timeout=120)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout == "ok\n"


def test_attributes_of_kernels_are_set_in_one_place():
    """which is the one that asks for the device (a static initializer would run on the first device only, and keep its error)"""
    at = [(os.path.basename(p), n) for p in sorted(glob.glob(os.path.join(CSRC, "*"))) if p.endswith((".hip", ".cpp", ".h"))
          for n, line in enumerate(open(p), 1) if re.search(r"\bhipFuncSetAttribute\s*\(", line)]
    assert [f for f, _ in at] == ["p8x_host.cpp"], at
