"""ouro_kv_attend's opt-in for more than 64 KiB of LDS (fp32 caches of heads
wider than 128) on every device that it runs on.  The runtime's answers come
from tests/cpp/two_devices.cpp, which prints each opt-in and launch; nothing
runs on a device."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

from ouroboros_amd import _lib

ROOT = Path(__file__).resolve().parents[1]
PROGRAM = """
import ctypes, sys
ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
from ouroboros_amd import _lib
lib = _lib.lib()
p = 1 << 20  # an address that nothing follows
cache = _lib.KvCacheDesc(p, p, p, 16 * 256, 256, 256, 8, 8, 16, 1, 256, _lib.DT_F32)
for device in (0, 0, 1, 0, 1):
    assert lib.ouro_init(device) == 0, lib.ouro_last_error()
    assert lib.ouro_kv_attend(ctypes.addressof(cache), None, p, 0, None, None, 0, None, p, None, 0, None, p, 0, None, _lib.DT_F32,
                              1, 1, 100, 1.0, p, None) == 0, lib.ouro_last_error()
"""


def test_each_device_opts_in(tmp_path):
    cc = shutil.which("g++")
    if cc is None or not _lib.LIB_PATH.exists():
        pytest.skip("no g++, or no library")
    so = tmp_path / "two_devices.so"
    build = subprocess.run([cc, "-O1", "-shared", "-fPIC", "-w", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                            str(ROOT / "tests" / "cpp" / "two_devices.cpp"), "-o", str(so)], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    r = subprocess.run([sys.executable, "-c", PROGRAM, str(so)], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    allowed, launches = set(), 0
    for line in r.stdout.splitlines():
        what, device, kernel, size = line.split()
        if what == "optin":
            allowed.add((device, kernel))
        elif int(size) > 60000:
            launches += 1
            assert (device, kernel) in allowed, r.stdout
    assert launches == 5, r.stdout
