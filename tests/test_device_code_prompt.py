"""The device code of the library of the operators around a prompt, as built: room for the waves that its attention lives from, nothing that
waits for a tile on its way to the LDS but where one is meant to, registers that stay registers."""
import os
import re
import shutil
import struct
import subprocess

import pytest

from adkv_amd.build import PROMPT_PATH
from test_device_code import _registers, early_sources, kernels
from test_lane_swaps import early_exchanges

LLVM = "/opt/rocm/llvm/bin"


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    if not os.path.exists(PROMPT_PATH) or not os.path.exists(f"{LLVM}/llvm-objdump"):
        pytest.skip("no library or no disassembler")
    d, found = tmp_path_factory.mktemp("code"), []
    subprocess.run([shutil.which("llvm-objcopy", path=LLVM), f"--dump-section=.hip_fatbin={d}/fat", PROMPT_PATH, f"{d}/copy"], check=True)
    fat = (d / "fat").read_bytes()
    for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", fat):
        p = m.start() + 32
        for _ in range(struct.unpack_from("<Q", fat, m.start() + 24)[0]):
            offset, size, n = struct.unpack_from("<QQQ", fat, p)
            if b"gfx950" in fat[p + 24:p + 24 + n]:
                (d / "code").write_bytes(fat[m.start() + offset:m.start() + offset + size])
                found.append([subprocess.run([f"{LLVM}/{tool}", *how, f"{d}/code"], check=True, capture_output=True, text=True).stdout
                              for tool, *how in (("llvm-objdump", "-d", "--no-show-raw-insn"), ("llvm-readelf", "--notes"))])
            p += 24 + n
    return found


def numbers(listings, name, *fields):
    """(kernel, fields of its description) of those whose names have `name` in them."""
    out = []
    for _, notes in listings:
        for kernel in re.split(r"\n  - (?=\.agpr_count)", notes)[1:]:
            full = re.search(r"\.name: +(\S+)", kernel)[1]
            if re.search(name, full):
                out.append((full, *(int(re.search(rf"\.{f}: +(\d+)", kernel)[1]) for f in fields)))
    return out


def test_registers_of_the_attention_leave_room_for_a_second_workgroup(listings):
    """Of 512 in steps of 8: two waves to a SIMD, four of 64 channels without a mask."""
    found = numbers(listings, r"1[01](many|some)_kernelILi[12]ELi(64|96|128)E", "vgpr_count")
    assert len(found) == 2 * 2 * 3 * 4 and not [f for f in found if f[1] > 256], found
    found = numbers(listings, r"11many_kernelILi[12]ELi64ELi0E", "vgpr_count")
    assert len(found) == 2 and not [f for f in found if f[1] > 128], found


def test_registers_stay_registers(listings):
    found = numbers(listings, r"_kernel", "private_segment_fixed_size", "vgpr_spill_count")
    assert len(found) > 100
    assert not [f for f in found if f[1] or f[2]], found


def test_nothing_waits_for_tiles_on_their_way_but_the_barriers(listings):
    """What the compiler does not know to have arrived it waits for at its first use, and with it for all that was asked for since."""
    seen = 0
    for text, _ in listings:
        for name, body in re.findall(r"^[0-9a-f]+ <(\S*11many_kernelILi[12]ELi\d+ELi0E\S*)>:\n(.*?)(?=^[0-9a-f]+ <|\Z)", text, re.S | re.M):
            code = re.findall(r"^\t(\S+)(?: +([^/\n]*?))? *//", body, re.M)
            products = [i for i, (op, _) in enumerate(code) if op.startswith("v_mfma")]
            barriers = [i for i, (op, _) in enumerate(code) if op == "s_barrier"]
            loop = range(barriers[-2], products[-1])          # two tiles behind a barrier each
            waits = [i for i in loop if code[i][0] == "s_waitcnt" and "vmcnt" in code[i][1]]
            assert len(barriers) == 3 and len(waits) == 1 and code[waits[0] + 1][0] == "s_barrier", (name, [code[i] for i in waits])
            seen += 1
    assert seen == 8


def test_distances_between_dependent_instructions(listings):
    """Matrix instructions and exchanges between lanes read what was written two wait states before; a swap is between two registers."""
    assert sum(t.count("\tv_mfma") for t, _ in listings) > 1000 and sum(t.count("_swap_b32") for t, _ in listings) > 100
    assert not [v for t, _ in listings for v in early_sources(t)][:5]
    assert not [v for t, _ in listings for v in early_exchanges(t)][:5]
    swaps = [(name, a) for t, _ in listings for name, code, _ in kernels(t, "v_permlane") for o, a, _ in code if o.endswith("_swap_b32_e32")]
    assert not [f for f in swaps if len(_registers(f[1])) != 2][:5]
