"""The build's check of kernels whose warps split the registers of the launch."""
import re

import pytest

from leanstream_b200 import build

LOG = """ptxas info    : Compiling entry function '_ZN3lsb1_chunk_attn_kernelINS_3F16ELi64ELb0EEEvv' for 'sm_100a'
    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads
ptxas info    : Used 168 registers, used 1 barriers
ptxas info    : Compiling entry function '_ZN3lsb1_chunk_attn_kernelINS_4BF16ELi128ELb1EEEvv' for 'sm_100a'
    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads
ptxas info    : Used {} registers, used 1 barriers
"""


def test_another_number_fails_the_build():
    build.check_registers("ls_attention_chunk.cu", LOG.format(128))
    build.check_registers("ls_append.cu", LOG.format(120))
    build.check_registers("ls_attention_chunk.cu", "")
    with pytest.raises(RuntimeError, match="BF16ELi128ELb1E.* 120 registers.* 128"):
        build.check_registers("ls_attention_chunk.cu", LOG.format(120))


def test_the_number_is_the_source_files():
    for src, (name, want) in build.REGISTERS.items():
        text = (build.CSRC / src).read_text()
        assert int(re.search(r"kRegs8 = (\d+)", text).group(1)) == want
        assert re.match(r"\w+", name).group(0)[:-1] in text
