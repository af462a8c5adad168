"""The bytes that opbench counts for the decode attention over an int8 cache."""
import numpy as np
import torch

import opbench
from oxide_b200.workloads import C3


def test_int8_decode_attention_counts_codes_scales_and_heads():
    c = C3()
    _, lens, _ = c.inputs()
    keys = int(np.sum(np.minimum(lens, c.keys)))
    for op, size in (("decode_attn_q8_bf16_c3", 2), ("decode_attn_q8_f32_c3", 4)):
        _, _, nb, shape = opbench.build(op, None, torch.device("cpu"))
        b, hq, hkv, m, d = shape
        # a scale of 4 bytes for 64 keys and head, in k and in v
        assert nb == keys * hkv * 2 * d + keys * hkv * 8 // 64 + 2 * b * hq * d * size
