"""Registers that a kernel keeps in memory are saved for all lanes (CPU only: the assembly of this library's kernels).

A spill's store that the compiler puts among the instructions of one side of a divergent branch saves the lanes of that
side alone; where the register is read back for all of them, the others get what was there before.  An address lost that
way faults the GPU.  So the sources whose kernels spill are looked through for such stores."""
import re
import subprocess

import pytest

from exactinfer_amd import build as B


def partial_stores(text):
    """Spill stores of each function at which the lanes may not all be on: those that follow, without the branch's end
    between, an instruction that turns lanes off."""
    found = []
    for name, body in re.findall(r"^(_Z\w+):.*?\n(.*?)^\.Lfunc_end", text, re.S | re.M):
        off = None
        for line in body.split("\n"):
            op = line.split(";")[0].strip()
            if re.match(r"s_or_b64 exec, exec|s_mov_b64 exec, -1", op):
                off = None
            elif re.match(r"s_\w*saveexec_b64|s_\w+_b64 exec,", op):
                off = op
            elif op.startswith("scratch_store") and off:
                found.append((name, op, off))
    return found


def test_what_is_looked_for():
    text = "_Z1kv:\n{}\ts_endpgm\n.Lfunc_end0:\n"
    save, half, end = "\tscratch_store_dword off, v1, off\n", "\ts_and_saveexec_b64 s[4:5], vcc\n", \
        "\ts_or_b64 exec, exec, s[4:5]\n"
    assert not partial_stores(text.format(save + half + end + save))
    assert len(partial_stores(text.format(half + save + end))) == 1
    other = "\ts_xor_b64 exec, exec, s[4:5]\n"
    assert len(partial_stores(text.format(half + "\ts_or_saveexec_b64 s[4:5], s[4:5]\n" + other + save + end))) == 1


@pytest.mark.parametrize("source", ["csrc/cache8.hip", "csrc/packed.hip", "csrc/prefill.hip"])
def test_spills_are_saved_for_all_lanes(source, tmp_path):
    out = tmp_path / "k.s"
    flags = [f for f in B.HIPCC_FLAGS if f != "-shared"]
    subprocess.run([B.hipcc(), *flags, "-S", "--offload-device-only", "-I", str(B.ROOT / "include"),
                    str(B.PKG / source), "-o", str(out)], check=True, capture_output=True, timeout=300)
    text = out.read_text()
    assert "s_endpgm" in text
    assert partial_stores(text) == []
