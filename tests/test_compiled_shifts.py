"""The compiled kernels hold no 64-bit shift whose amount lies in the last vector register of a wave's allocation: it takes
its amount from the registers that follow, another wave's, and gives wrong values at times."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from odie_amd import _lib

TOOLS = Path('/opt/rocm/llvm/bin')
GRANULE = 8         # registers that a wave is given together
SHIFT = re.compile(r'\bv_(?:lshlrev_b64|lshrrev_b64|ashrrev_i64)\S* v\[\d+:\d+\], v(\d+),')


def _registers(code):
    symbols = subprocess.run([TOOLS / 'llvm-readelf', '-s', '-W', code], capture_output=True, text=True, check=True).stdout
    return {name: int(value, 16) for value, name in re.findall(r'\d+: ([0-9a-f]+) .* (\S+)\.num_vgpr$', symbols, re.M)}


def _shifts_by_the_last(listing, registers):
    found, kernel = [], None
    for line in listing:
        start = re.match(r'[0-9a-f]+ <(.+)>:', line)
        if start:
            kernel = start.group(1)
            continue
        shift = SHIFT.search(line)
        if shift and (int(shift.group(1)) + 1) % GRANULE == 0 and int(shift.group(1)) + 1 >= registers.get(kernel, 0):
            found.append((kernel, line.strip()))
    return found


def test_the_scan_itself():
    listing = ['0000000000000100 <one>:', '\tv_lshlrev_b64 v[28:29], v31, v[2:3]', '\tv_lshlrev_b64 v[28:29], 3, v[2:3]',
               '\tv_lshrrev_b64 v[28:29], v30, v[2:3]', '0000000000000200 <two>:', '\tv_ashrrev_i64 v[4:5], v31, v[2:3]']
    assert _shifts_by_the_last(listing, {'one': 32, 'two': 40}) == [('one', 'v_lshlrev_b64 v[28:29], v31, v[2:3]')]


def test_no_shift_by_the_last_register(tmp_path):
    if not (TOOLS / 'llvm-objdump').exists() or not Path(_lib.LIBRARY).exists():
        pytest.skip('needs the built library and ROCm\'s llvm-objdump')
    shutil.copy(_lib.LIBRARY, tmp_path / 'library.so')
    subprocess.run([TOOLS / 'llvm-objdump', '--offloading', 'library.so'], cwd=tmp_path, capture_output=True, check=True)
    codes = sorted(tmp_path.glob('*gfx950*'))
    assert codes
    shifts = 0
    for code in codes:
        listing = subprocess.run([TOOLS / 'llvm-objdump', '-d', '--no-show-raw-insn', code], capture_output=True, text=True,
                                 check=True).stdout.splitlines()
        registers = _registers(code)
        assert registers
        shifts += sum(SHIFT.search(line) is not None for line in listing)
        assert _shifts_by_the_last(listing, registers) == []
    print('%d shifts by a register' % shifts)
