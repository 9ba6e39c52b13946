"""The matrix-core kernels of packed query tokens read no MFMA result sooner after a branch than
the compiler allows on straight-line paths, and their exchange between the halves of a wave is
emitted (see isa_hazards.py and test_isa_hazards.py). Compiles them to assembly with the library's
own flags; no GPU needed."""

from __future__ import annotations

import shutil
import subprocess
from collections import defaultdict
from concurrent.futures import ThreadPoolExecutor

import pytest

from tests import isa_hazards
from vllm_fastdecoder_amd import build

SOURCES = ["prefill_mm_f16.hip", "prefill_mm_bf16.hip", "prefill_mm_f32.hip"]


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    if shutil.which(build.hipcc()) is None:
        pytest.skip("hipcc not available")
    tmp = tmp_path_factory.mktemp("isa")

    def one(src):
        out = tmp / (src + ".s")
        cmd = [build.hipcc(), *build.HIPCC_FLAGS, *build.SOURCE_FLAGS.get(src, []),
               "--cuda-device-only", "-S", str(build.CSRC / src), "-o", str(out)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        assert res.returncode == 0, res.stderr[-2000:]
        return out.read_text()

    with ThreadPoolExecutor(max_workers=len(SOURCES)) as pool:
        return dict(zip(SOURCES, pool.map(one, SOURCES)))


@pytest.mark.parametrize("src", SOURCES)
def test_no_mfma_result_read_early_across_a_branch(asm, src):
    gaps = [g for name, ins, labels in isa_hazards.kernels(asm[src])
            for g in isa_hazards.mfma_read_gaps(name, ins, labels)]
    assert gaps, "no MFMA result reads found: the parser no longer matches the assembly"
    straight = defaultdict(lambda: 1 << 30)
    for g in gaps:
        if not g.via_branch:
            straight[g.mfma] = min(straight[g.mfma], g.wait_states)
    short = [g for g in gaps if g.via_branch and g.mfma in straight
             and g.wait_states < straight[g.mfma]]
    assert not short, "\n".join(
        f"{g.kernel}: {g.mfma} read by {g.reader} after {g.wait_states} wait states across "
        f"a branch (straight-line minimum {straight[g.mfma]})" for g in short[:10])


@pytest.mark.parametrize("src", SOURCES)
def test_the_halves_of_a_wave_exchange_their_maximum_and_sum(asm, src):
    names = [(name, ins) for name, ins, _ in isa_hazards.kernels(asm[src])
             if "prefill_mm_kernel" in name]
    assert names, "no kernels found in the assembly"
    missing = [name for name, ins in names
               if not any(op.startswith("v_permlane32_swap") for op, _ in ins)]
    assert not missing, missing
