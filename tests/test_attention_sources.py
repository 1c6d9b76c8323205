"""What the compiler is told about the kernels' inline assembly."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "spmm-research_amd" / "csrc"


def test_assembly_names_m0_where_it_writes_it():
    """Otherwise nothing keeps its own uses of m0 (LDS addressing, register indexing) apart from these."""
    found = 0
    for f in sorted(CSRC.glob("attn_*")) + [CSRC / "matvec_q4.hip"]:
        for text in re.findall(r"asm volatile\((.*?)\);", f.read_text(), re.S):
            if re.search(r"s_mov_b32 m0", text):
                found += 1
                assert '"m0"' in text.split("::")[-1], (f.name, text)
    assert found == 2
