"""CPU tests of the latent kernels' host-side arithmetic, compiled from the library's own headers."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_deal_and_joinable_units(tmp_path):
    """Entries of units that a CTA never wrote may hold anything: only pieces of the launch's CTAs are joined."""
    exe = str(tmp_path / "test_latent_deal")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I" + os.path.join(ROOT, "vulcan_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "test_latent_deal.cpp"), "-o", exe], check=True, capture_output=True, text=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "0 failures" in r.stdout, r.stdout + r.stderr
