"""The compiler's resource remarks of the training operators' kernels (csrc/train/*.ru.txt): none uses scratch memory, and
those that share a compute unit two at a time keep to half of its registers and shared memory."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))
import kernel_resources as KR  # noqa: E402

TRAIN = os.path.join(KR.CSRC, "train")
SRCS = ["r3_logprob", "r3_ortho"]


@pytest.fixture(scope="module")
def rows():
    if any(not os.path.exists(os.path.join(TRAIN, s + ".ru.txt")) for s in SRCS):
        subprocess.run(["make", "-C", KR.CSRC, "-j8", "all"], check=True, stdout=subprocess.DEVNULL)
    got = KR.collect(TRAIN)
    assert {r["file"] for r in got} == {s + ".hip" for s in SRCS}
    return got


def test_no_scratch(rows):
    assert len(rows) > 60
    assert not [(r["short"], r["scratch"]) for r in rows if r["scratch"]]


def test_two_workgroups_of_a_product_fit_a_compute_unit(rows):
    got = [r for r in rows if any(k in r["short"] for k in ("ortho_gram", "ortho_square", "ortho_apply"))]  # (mangled or not)
    assert len(got) >= 17
    for r in got:
        assert r["vgpr"] <= 256 and r["agpr"] == 0 and r["occupancy"] >= 2, r["short"]
        eight = "Core64ILi8E" in r["name"]  # (eight wavefronts: one workgroup)
        assert r["lds"] <= (160 * 1024 if eight else 80 * 1024), (r["short"], r["lds"])
