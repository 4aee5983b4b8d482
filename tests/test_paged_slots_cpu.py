"""The parts of items lie in the workspace in slots that the kernels store to in words of 32 bytes: every slot begins on one, whatever the heads of a
key head make of an item's rows.  (Checked by the sizes that the library asks for: an odd slot off 32 bytes would be a misaligned store.)"""
import pytest

from test_paged_cpu import _args as paged
from test_prompt_cpu import _args as prompt

CTAS, RECORDS = 148, 148 * 28 + -(148 * 28) % 256            # one record of seven ints a CTA, then two slots a CTA


@pytest.mark.parametrize("c", [64, 128])
@pytest.mark.parametrize("N", [1, 7, 100, 20000])
def test_slots_begin_on_32_bytes(c, N):
    from kch_b200 import _lib
    lib = _lib.load()
    for G in range(1, 260):
        sizes = [int(lib.kch_prompt_attend_workspace_bytes(prompt(_lib, N=N, nh=G, n_kv=1, c=c, ld_q=G * c, ld_k=c, ld_v=c)))]
        for kind in (1, 2, 3, 4):
            sizes.append(int(lib.kch_paged_attend_workspace_bytes(paged(_lib, kind=kind, N=N, nh=G, n_kv=1, c=c, ld_q=G * c))))
        for size in sizes:
            slot = (size - RECORDS) // (2 * CTAS)
            assert (size - RECORDS) % (2 * CTAS) == 0 and slot >= 4 * (c + 2) * min(N * G, 8) and slot % 32 == 0, f"{G} heads of a key head: slots of {slot} bytes"
