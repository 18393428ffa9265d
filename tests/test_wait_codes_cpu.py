"""The bounded waits of the tensor-core kernels record a code each: a code names one wait of one file."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_wait_codes_name_one_wait():
    seen = {}
    for path in sorted(glob.glob(os.path.join(ROOT, "csrc", "*.cu"))):
        with open(path) as f:
            for code in re.findall(r"mbar_wait\([^;{]*?, (\d+)\)", f.read()):
                seen.setdefault(int(code), []).append(os.path.basename(path))
    assert len(seen) > 20 and {"gemm_sm100.cu", "wgrad_sm100.cu", "attention_sm100.cu"} <= {p for v in seen.values() for p in v}
    shared = {code: paths for code, paths in seen.items() if len(set(paths)) > 1}
    assert not shared, shared
