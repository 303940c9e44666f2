"""Set-ups that belong to a device (a kernel's shared memory limit) are made on each device that a process
uses, and made again after they failed."""
import os
import re
import shutil
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "openasr_b200", "csrc")
CXX = shutil.which("g++", path="/usr/bin") or shutil.which("g++") or "g++"

SOURCE = r"""
#include <cstdio>
#include <initializer_list>
#include "once_per_device.h"
int main() {
    oasr::OncePerDevice once, other;
    int n = 0, status = 0;
    auto set_up = [&] { ++n; return status; };
    for (int device : {0, 0, 1, 0, 1, 63, 63, 0}) once(device, set_up);
    std::printf("%d ", n);
    other(0, set_up);
    std::printf("%d ", n);
    status = 7;
    std::printf("%d ", once(2, set_up));
    status = 0;
    std::printf("%d ", once(2, set_up));
    once(2, set_up), once(64, set_up), once(64, set_up);
    std::printf("%d", n);
}
"""


def test_once_on_each_device(tmp_path):
    (tmp_path / "once.cpp").write_text(SOURCE)
    subprocess.run([CXX, "-std=c++17", "-I", CSRC, str(tmp_path / "once.cpp"), "-o", str(tmp_path / "once")], check=True)
    assert subprocess.run([str(tmp_path / "once")], check=True, capture_output=True, text=True).stdout == "3 4 7 0 8"


def test_no_kernel_attribute_is_set_once_per_process():
    """every file that raises a kernel's limit does so per device (dgemv.cu keeps its own record)"""
    for f in sorted(os.listdir(CSRC)):
        if f.endswith(".cu") and f != "dgemv.cu":
            text = open(os.path.join(CSRC, f)).read()
            calls = len(re.findall(r"cudaFuncSetAttribute\(", text))
            assert len(re.findall(r"static OncePerDevice \w+;", text)) == calls, f
            assert not re.search(r"static std::atomic<bool>", text), f
