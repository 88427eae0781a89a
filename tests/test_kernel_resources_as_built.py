"""Register budgets of the kernels as they are built: the compile commands come from the Makefile, with its flags (CPU:
hipcc cross-compiles for gfx950 and reports per-kernel resources)."""
import os
import re
import shlex
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC) and shutil.which("hipcc") is None, reason="no hipcc")


def command(target):
    """The Makefile's command for one object file."""
    out = subprocess.run(["make", "-n", "-B", target], cwd=ROOT, capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stderr
    line, = [c for c in out.stdout.splitlines() if " -c " in c]
    return shlex.split(line)


@pytest.fixture(scope="module")
def scratch(tmp_path_factory):
    """source -> {kernel: bytes of scratch memory per lane}; the sources are compiled side by side."""
    to, running = tmp_path_factory.mktemp("resources"), {}
    for source in ("conv_patch", "groupnorm", "linear", "distill"):
        cmd = command("cvae_gan_amd/csrc/%s.o" % source)
        cmd[cmd.index("-o") + 1] = str(to / (source + ".o"))
        log = open(to / (source + ".log"), "w")
        running[source] = subprocess.Popen(cmd + ["--offload-device-only", "-Rpass-analysis=kernel-resource-usage"], cwd=ROOT, stderr=log)
    found = {}
    for source, p in running.items():
        rc, text = p.wait(timeout=900), (to / (source + ".log")).read_text()
        assert rc == 0, text[-2000:]
        found[source], name = {}, None
        for line in text.splitlines():
            m = re.search(r"Function Name: (\S+)", line)
            if m:
                name = m.group(1)
            m = re.search(r"ScratchSize \[bytes/lane\]: (\d+)", line)
            if m and name:
                found[source][name] = int(m.group(1))
    return found


def test_the_flags():
    """Every HIP compile leaves the packed f32 instructions out."""
    for target in ("conv_patch", "igemm", "elementwise", "api", "groupnorm", "linear", "distill"):
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in " ".join(command("cvae_gan_amd/csrc/%s.o" % target))
    out = subprocess.run(["make", "-n", "-B", "timing"], cwd=ROOT, capture_output=True, text=True, timeout=60)
    for line in out.stdout.splitlines():
        if ".hip" in line and "hipcc" in line:
            assert "-packed-fp32-ops" in line, line


def test_bf16_convolution_kernels_do_not_spill(scratch):
    hot = re.compile("patch_fwdIDF16b|patch_wgrad9|patch_dgrad_s2IDF16b|patch_wgradIDF16b|lowk_fwd")
    found = {n: b for n, b in scratch["conv_patch"].items() if hot.search(n)}
    assert len(found) >= 20 and not any(found.values()), {n: b for n, b in found.items() if b}


def test_linear_and_distillation_kernels_do_not_spill(scratch):
    for source, least in (("linear", 15), ("distill", 30)):
        found = scratch[source]
        assert len(found) >= least and not any(found.values()), {n: b for n, b in found.items() if b}


def test_group_norm_kernels_spill_only_in_the_widest_forward_form(scratch):
    """gn_fwd_tile at its widest (128 registers: 16 bf16 or 8 f32 chunks a thread) keeps up to 68 bytes per lane in scratch
    memory, mostly gamma and beta; every other kernel none."""
    found = scratch["groupnorm"]
    wide = re.compile("gn_fwd_tileI(DF16bLi.ELi16E|fLi.ELi8E)")
    assert sum(bool(wide.search(n)) for n in found) == 8
    assert not {n: b for n, b in found.items() if b > (68 if wide.search(n) else 0)}
