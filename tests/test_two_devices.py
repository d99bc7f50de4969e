"""Set-up calls of the block-scaled cache in a process with two devices: the library's host sources
over a pretend runtime (two_devices.cpp), since one device shows nothing of it."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "eyebrowse_amd", "csrc")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


def test_a_cache_is_made_on_its_device(tmp_path):
    exe = str(tmp_path / "two_devices")
    sources = [os.path.join(CSRC, f) for f in ("eb_runtime.cpp", "eb_nn.cpp", "eb_quant.cpp")]
    # (the kernels' launchers, which no call here reaches, are left out)
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROCM, "include"),
                    "-I", CSRC, "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "two_devices.cpp"),
                    *sources, "-Wl,--unresolved-symbols=ignore-all", "-o", exe], check=True, stderr=subprocess.DEVNULL)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
