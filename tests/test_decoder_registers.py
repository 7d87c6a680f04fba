"""CPU test of the registers that the compiler spilled in the attention of few rows - it takes every decode step - and in the norm: no more bytes (stores, loads) than the
figures below, none where there is no figure."""
import re
from pathlib import Path

import pytest

BUILD = Path(__file__).resolve().parents[1] / "dinoml_v2_b200" / "build"
FEW = "attention_few_kernelILi{}ENS1_5ShapeILi{}ELi{}ELi{}EEE"      # cache type (int8, e4m3), head size, tiles of eight rows, terms (float32: two)
NORM = "rms_norm_kernelI{}{}Li8ELb{}ELi{}ELi{}ELb{}EEE"             # activations, weights, wide accesses, rounds, threads, Q8_0
BF16, F16, F32 = "13__nv_bfloat16", "6__half", "f"
SAME = "S2_"                                                        # weights of the activations' type
CEILINGS = {
    "ptxas_kv_attention_few_int8.log": {
        FEW.format(1, 64, 2, 2): (20, 48), FEW.format(1, 128, 1, 1): (8, 8), FEW.format(1, 128, 1, 2): (12, 12), FEW.format(1, 128, 2, 1): (24, 44),
        FEW.format(1, 128, 2, 2): (48, 68), FEW.format(1, 256, 1, 1): (60, 84), FEW.format(1, 256, 1, 2): (60, 84),
    },
    "ptxas_kv_attention_few_e4m3.log": {
        FEW.format(2, 64, 2, 1): (20, 40), FEW.format(2, 128, 1, 1): (12, 16), FEW.format(2, 128, 1, 2): (20, 28), FEW.format(2, 128, 2, 1): (24, 44),
        FEW.format(2, 128, 2, 2): (72, 96), FEW.format(2, 256, 1, 1): (64, 88), FEW.format(2, 256, 1, 2): (64, 88),
    },
    "ptxas_rms_norm.log": {
        # rows of more than 8192 16-bit values, and to Q8_0 of more than 4096 with bfloat16 weights
        **{NORM.format(t, w, 1, 4, 1024, 1): (124, 60) for t in (BF16, F16) for w in (SAME, F32)},
        **{NORM.format(t, w, 0, 4, 1024, 1): (60, 40) for t in (BF16, F16) for w in (SAME, F32)},
        **{NORM.format(F16, w, 1, 4, 1024, 0): (8, 4) for w in (SAME, F32)},
        NORM.format(BF16, SAME, 1, 4, 1024, 0): (40, 20), NORM.format(BF16, F32, 1, 4, 1024, 0): (24, 12), NORM.format(BF16, SAME, 1, 2, 512, 1): (28, 44),
    },
}


@pytest.mark.parametrize("log", sorted(CEILINGS))
def test_spills_stay_below_their_ceilings(log):
    path = BUILD / log
    if not path.exists():
        pytest.skip("no ptxas log: the library was not built in this tree")
    entries = re.findall(r"Compiling entry function '(\S+)'.*?\n.*?\n\s*\d+ bytes stack frame, (\d+) bytes spill stores, (\d+) bytes spill loads", path.read_text())
    assert len(entries) >= len(CEILINGS[log])
    for part in CEILINGS[log]:
        assert sum(part in name for name, _, _ in entries) == 1, part
    for name, stores, loads in entries:
        most = next((c for part, c in CEILINGS[log].items() if part in name), (0, 0))
        assert int(stores) <= most[0] and int(loads) <= most[1], (name, stores, loads, most)
