"""The digest that says whether a measured row of the step's memory traffic is current goes by
the sources of the step's kernels, and by those alone.  CPU only."""
import shutil

import pytest

import bench
from tatara_amd import build


@pytest.fixture
def sources(tmp_path, monkeypatch):
    """A copy of the kernel sources that may be changed."""
    shutil.copytree(build.CSRC, tmp_path / "csrc")
    monkeypatch.setattr(build, "CSRC", tmp_path / "csrc")
    return tmp_path / "csrc"


def test_what_a_step_is_built_from():
    names = {f.name for f in build.step_sources()}
    assert {"trainer.hip", "simple_trainer.hip", "ft_kernels.hip", "dense_kernels.hip", "simple_kernels.hip",
            "binsort.hip", "psv_kernels.hip", "optim.hpp", "loss.hpp", "common.hpp"} <= names
    assert not {"muon_kernels.hip", "norm_kernels.hip", "gate_kernels.hip"} & names


def test_other_operators_leave_it_alone(sources):
    before = build.step_digest()
    for name in ("muon_kernels.hip", "gate_kernels.hip", "elem.hpp"):
        (sources / name).write_text("// another operator\n")
    (sources / "more_kernels.hip").write_text("// one more\n")
    assert build.step_digest() == before
    (sources / "optim.hpp").write_text((sources / "optim.hpp").read_text() + "// changed\n")
    assert build.step_digest() != before


def test_traffic_rows_name_such_a_digest():
    """The same for all rows, in the form that the digest has."""
    digests = set()
    for workload, kernel in (("ls1536", "ft_grad_scan_kernel"), ("ls1536_mixed", "ft_grad_mfma_kernel"),
                             ("ls768", "ft_grad_scan_kernel"), ("simple", "ft_forward")):
        traffic, commit, digest = bench.hbm_traffic(workload, kernel)
        assert traffic and commit, workload
        digests.add(digest)
    assert len(digests) == 1 and len(digests.pop()) == len(build.step_digest())
