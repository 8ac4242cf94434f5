"""The library holds no kernel of the choice that no call reaches."""
from pathlib import Path

import pytest

from odie_amd import _lib


def test_rows_read_once_a_choice_are_fp32():
    """16-bit rows of the most experts, 32768, stay in registers."""
    if not Path(_lib.LIBRARY).exists():
        pytest.skip('needs the built library')
    code = Path(_lib.LIBRARY).read_bytes()
    names = [name for name in (b'choose_long_kernelIfE', b'choose_long_kernelE', b'choose_long_kernelIDF16') if name in code]
    assert names and b'choose_long_kernelIDF16' not in names
