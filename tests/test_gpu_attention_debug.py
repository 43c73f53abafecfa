"""The attention kernels under the debug build (LDS, outputs and workspaces filled
with NaN first), each case a test of another file run again."""
import pytest
import torch

from pseudobrain_amd import _lib
from tests import test_gpu_paged_attention as paged
from tests import test_gpu_window_attention as window

pytestmark = pytest.mark.gpu

CASES = {
    "lengths": lambda: window.test_lengths_windows_and_sinks(200, 100, 70, torch.bfloat16),
    "groups": lambda: window.test_head_groups(7, 1),
    "groups beyond a tile": lambda: window.test_head_groups(40, 1),
    "256 wide": lambda: window.test_widths_and_types(256, torch.bfloat16),
    "256 wide, float32": lambda: window.test_widths_and_types(256, torch.float32),
    "float16": lambda: window.test_widths_and_types(128, torch.float16),
    "rows that see nothing": lambda: window.test_queries_and_keys_of_different_lengths(90, 40, 50, 4),
    "packed": lambda: window.test_packed_sequences(torch.bfloat16, 128),
    "packed queries and keys": window.test_packed_queries_and_keys,
    "split walks": lambda: window.test_long_walks_are_split(torch.bfloat16),
    "pages": lambda: paged.test_pages_windows_and_lengths(40, 5, 7),
    "drafts": lambda: paged.test_head_groups_and_drafts(24, 8, 4),
    "joined parts": paged.test_long_contexts_are_split_and_joined,
    "decode, 256 wide": lambda: paged.test_widths_and_types(256, torch.bfloat16),
}


@pytest.mark.parametrize("case", CASES)
def test_under_the_debug_build(case):
    with _lib.debug_library():
        CASES[case]()


SINKS = {
    "short and long sequences": lambda: window.test_sinks_of_packed_short_and_long_sequences(2, 4),
    "short and long sequences, many sinks": lambda: window.test_sinks_of_packed_short_and_long_sequences(1, 70),
    "parts beside the sinks'": lambda: window.test_sinks_of_a_long_packed_call(1),
}


@pytest.mark.parametrize("case", SINKS)
def test_sinks_under_the_debug_build(case):
    """A part of the sinks' that is joined but was not written shows as NaN."""
    with _lib.debug_library():
        SINKS[case]()
