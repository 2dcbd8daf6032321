"""The numbers that kernels leave where a bounded wait ran out, on the CPU: each is named by CudaOps.check_errors, and a name's numbers belong to its kernels alone."""
import os
import re

import pytest
import torch

from mini_inference_b200.ops import CudaOps
from mini_inference_b200.ops.build import CSRC

OWNERS = {"gemm_stream": {"gemm_stream.cu"}, "attention": {"attention_prefill_tc.cu", "attention_decode_mma.cu"}, "recurrences eight tokens at a time": {"state_octets.cu"},
          "gemm_tc2": {"gemm_tc2.cu"}, "grouped expert product": {"moe_grouped_tc.cu"}, "delta rule and constant decay in chunks": {"state_chunks.cu", "gated_delta.cu", "gated_delta_chunk.cu"},
          "float32 product": {"gemm_f32_tc.cu"}, "channel decays in chunks": {"channel_chunks.cu"}, "attention over shared prefixes": {"attention_shared_tc.cu"}}


def message(code):
    me = CudaOps.__new__(CudaOps)
    me._stream_error, me._tc2_counters = torch.tensor([code], dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError) as e:
        me.check_errors()
    assert int(me._stream_error) == 0
    me.check_errors()                                              # told once
    return str(e.value)


def test_every_code_has_one_name():
    text = message(5)
    names = {name.strip(): range(int(a), int(b) + 1) for a, b, name in re.findall(r"(\d+)-(\d+) ([^,)]+)", text)}
    assert set(names) == set(OWNERS)
    files = {}
    for file in sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))):
        with open(os.path.join(CSRC, file)) as f:
            codes = {int(c) for c in re.findall(r"atomicExch\((?:error_word|error), (\d+)\)", f.read())}
        if codes:
            files[file] = codes
    assert set(files) == set().union(*OWNERS.values())
    for file, codes in files.items():
        for code in codes:
            assert [name for name, span in names.items() if code in span] == [name for name, own in OWNERS.items() if file in own], (file, code)
