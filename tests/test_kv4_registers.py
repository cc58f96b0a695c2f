"""What the 4-bit attention's kernels ask of a SIMD's 512 vector registers (the code objects' own metadata; no GPU)."""
import re

from test_kernel_registers import kernels


def test_no_spills_and_the_waves_a_simd(tmp_path):
    """None spills; prompts of heads of 64 have three waves a SIMD (168 registers), single rows of heads of 64 and up to
    four a group four (128), and every chunk form, heads of 256 among them, two (256)."""
    found = {}
    for name, (registers, spilled) in kernels("attention_kv4", tmp_path).items():
        assert spilled == 0, name
        form = re.search(r"attention_kv4(_row)?_kernelI((?:L[ij]\d+E)+)E", name)
        if form:
            found[(form.group(1) or "",) + tuple(int(x) for x in re.findall(r"L[ij](\d+)E", form.group(2)))] = registers
    assert len(found) == 39
    assert found["", 2, 2, 2, 4] <= 168 and found["", 2, 2, 4, 4] <= 168
    assert found["_row", 2, 1, 4] <= 128 and found["_row", 2, 1, 8] <= 128
    assert all(registers <= 256 for form, registers in found.items() if form[0] == "")
