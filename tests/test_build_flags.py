"""How the HIP sources are compiled: every file without packed fp32 arithmetic, none of which is spelled out either."""
import glob
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "evfly_amd", "csrc")


def test_every_file_is_compiled_without_packed_fp32():
    said = subprocess.run(["make", "-n", "-B", "-C", CSRC], capture_output=True, text=True, check=True).stdout
    lines = {re.search(r"-c (\w+)\.hip", line).group(1): line for line in said.splitlines() if " -c " in line}
    assert sorted(lines) == sorted(os.path.basename(p)[:-4] for p in glob.glob(os.path.join(CSRC, "*.hip")))
    for name, line in lines.items():
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, name


def test_no_source_spells_packed_fp32():
    for path in glob.glob(os.path.join(CSRC, "*.h*")):
        for i, line in enumerate(open(path), 1):
            assert not re.search(r"v_pk_(add|mul|fma)_f32", line), f"{path}:{i}"


def test_no_source_queues_a_memset():
    """A captured hipMemsetAsync node may go wrong on replays: memory is filled by a kernel."""
    for path in glob.glob(os.path.join(CSRC, "*.h*")):
        code = re.sub(r"//[^\n]*", "", open(path).read())
        assert "hipMemsetAsync" not in code, path
