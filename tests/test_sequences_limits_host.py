"""What attention over a paged cache asks for in memory, from the entry point that says so."""
import ctypes
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def bytes_of():
    from qwen_image_edit_streamdiffusion_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        import subprocess
        subprocess.run(["make", "-C", os.path.join(ROOT, "qwen_image_edit_streamdiffusion_amd", "csrc"), "-j8"],
                       check=True, capture_output=True)
    lib = _lib.load()

    def get(tokens, seqs, heads, kv_heads, head_dim, width, page):
        n = ctypes.c_int64(-1)
        assert lib.qie_attention_paged_workspace(tokens, seqs, heads, kv_heads, head_dim, width, page, ctypes.byref(n)) == 0
        return n.value
    return get


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(28, 4, 128), (40, 40, 128), (64, 8, 128), (16, 16, 80), (8, 8, 64), (20, 1, 128)])
@pytest.mark.parametrize("table", [1 << 11, 1 << 14, 1 << 17, 1 << 20, 1 << 26])
def test_workspace_is_bounded(bytes_of, heads, kv_heads, head_dim, table):
    """The parts of cut rows take 256 MiB at most, however wide the table and however many the rows. The lengths may be
    short: what they would need is not known to the host."""
    for seqs in (1, 3, 32, 128, 1000):
        for new in (1, 4, 16, 17, 33, 64, 65, 100, 300, 1500):
            if seqs * new * heads <= 1 << 30:
                assert 0 <= bytes_of(seqs * new, seqs, heads, kv_heads, head_dim, table // 64, 64) <= 256 << 20, (seqs, new)


def test_few_rows_over_a_long_table_are_still_cut(bytes_of):
    """A bound that left no cut would put a single token's 32768 keys on four work-groups."""
    assert bytes_of(1, 1, 28, 4, 128, 512, 64) >= 28 * 8 * 130 * 4
    assert bytes_of(128, 32, 28, 4, 128, 512, 64) > 0 and bytes_of(1 << 20, 1, 1, 1, 128, 1 << 18, 64) >= 0


@pytest.mark.parametrize("new,table", [(2200, 24000), (2340, 24000), (2340, 1 << 17), (4500, 24000), (4600, 12000)])
def test_one_sequence_whose_blocks_fill_the_chip_is_not_cut_in_chunks(bytes_of, new, table):
    """It takes equal shares as any other: two blocks of 256 rows of parts for each of 256 work-groups."""
    assert bytes_of(new, 1, 28, 4, 128, table // 64, 64) == 256 * 2 * 256 * 130 * 4
