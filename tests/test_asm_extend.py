"""The extension attention's second product is an inline-asm MFMA with its sums in
AGPRs (`v_mfma_f32_32x32x16_bf16 a[...], v[...], v[...], a[...]`). The compiler does not
see into asm: it adds no wait states between a VALU write of an operand and the
product (two are needed), and none between the product and a VALU read of its sums
(18 for 16 passes; the source ends every run of products with 24). This test compiles
the source with the library's own flags and scans the gfx950 assembly: no vector
instruction writes an operand within two wait states before such a product, no
instruction but another such product touches sums before the waits behind them, and
the loops over tiles use no scratch memory. The scanner itself is checked on
hand-written sequences."""
import re
import subprocess
import sys
from pathlib import Path

REPO = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(REPO / "gemma.c_amd"))
from gemma_kv import build as kb  # noqa: E402

REG = re.compile(r"\b([av])(?:\[(\d+):(\d+)\]|(\d+)\b)")
PRODUCT = re.compile(r"^\s*v_mfma_\w+\s+a\[")
OPERAND_WAITS, RESULT_WAITS = 2, 18


def registers(text):
    return {(m.group(1), i) for m in REG.finditer(text)
            for i in range(int(m.group(2) or m.group(4)), int(m.group(3) or m.group(4)) + 1)}


def scan(lines):
    """(line number, instruction, why) of every hazard. Each wait state is one
    instruction; `s_nop n` is n + 1. A label is reached from elsewhere too: behind one,
    the way that falls through is looked at, and sums count as in flight as before."""
    bad = []
    written = []   # [wait states ago, vector registers] of the newest VALU writes
    flying = {}    # AGPR -> wait states since its product
    for no, raw in enumerate(lines, 1):
        line = raw.split(";")[0].strip()
        if not line or line.endswith(":") or line.startswith("."):
            continue
        name, _, rest = line.partition(" ")
        operands = rest.split(",")
        if PRODUCT.match(line):
            used = registers(",".join(re.findall(r"v\[\d+:\d+\]|\bv\d+", rest)))
            if any(ago < OPERAND_WAITS and regs & used for ago, regs in written):
                bad.append((no, line, "an operand was just written"))
        else:
            for reg in registers(rest):
                if flying.get(reg, RESULT_WAITS) < RESULT_WAITS:
                    bad.append((no, line, "sums are still being written"))
                    break
        waits = int(rest, 0) + 1 if name == "s_nop" else 1
        written = [(ago + waits, regs) for ago, regs in written if ago + waits < OPERAND_WAITS]
        flying = {reg: ago + waits for reg, ago in flying.items() if ago + waits < RESULT_WAITS}
        if PRODUCT.match(line):
            flying.update({reg: 0 for reg in registers(operands[0])})
        elif name.startswith("v_") and not name.startswith("v_cmp"):
            swap = name.startswith(("v_swap", "v_permlane16_swap", "v_permlane32_swap"))
            written.append((0, registers(rest if swap else operands[0])))
        if name == "s_endpgm":
            written, flying = [], {}
    return bad


def test_scanner_on_hand_written_sequences():
    product = "v_mfma_f32_32x32x16_bf16 a[0:15], v[40:43], v[32:35], a[0:15]"
    assert scan([product, product]) == []
    assert scan(["v_mov_b32_e32 v40, v1", "s_nop 1", product]) == []
    assert scan(["v_mov_b32_e32 v44, v1", product]) == []
    assert len(scan(["v_mov_b32_e32 v40, v1", "s_nop 0", product])) == 1
    assert len(scan(["v_permlane32_swap_b32_e32 v1, v33", product])) == 1
    assert len(scan([product, "s_nop 15", "v_accvgpr_read_b32 v1, a3"])) == 1
    assert scan([product, "s_nop 15", "s_nop 7", "v_accvgpr_read_b32 v1, a3"]) == []
    assert scan([product, "v_accvgpr_read_b32 v1, a16"]) == []


def test_second_products_and_scratch(tmp_path):
    out = tmp_path / "extend_rows.s"
    cmd = [kb.HIPCC, *kb.HIP_FLAGS, *kb.EXTRA_FLAGS["extend_rows"], "--cuda-device-only", "-S",
           str(kb.CSRC_DIR / "extend_rows.hip"), "-o", str(out)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-2000:]
    lines = out.read_text().splitlines()
    assert sum(bool(PRODUCT.match(l)) for l in lines) >= 32
    bad = scan(lines)
    assert bad == [], bad[:5]
    # Blocks of the loops over tiles, by the compiler's notes behind their labels.
    depth, inner, spilled = 0, 0, []
    for no, line in enumerate(lines, 1):
        if re.match(r"^\.LBB\d+_\d+:|^; %bb\.\d+:", line):
            depth = 0
        note = re.search(r"Depth=(\d+)", line)
        if note and (line.lstrip().startswith(";") or line.startswith(".LBB")):
            depth = max(depth, int(note.group(1)))
        if depth >= 2:
            inner += bool(PRODUCT.match(line))
            if re.match(r"^\s*scratch_", line):
                spilled.append((no, line.strip()))
    assert inner >= 32, "the loops over tiles were not found"
    assert spilled == [], spilled[:5]
