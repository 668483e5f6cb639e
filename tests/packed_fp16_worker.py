"""Child process of tests/test_packed_fp16_gpu.py (test infrastructure): the packed-sequence operators on the IEEE-half
flavour of the library (MELGPT_HALF=fp16), by the same checks against 64-bit definitions that the bfloat16 flavour passes."""
import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
for p in (os.path.dirname(HERE), HERE):
    sys.path.insert(0, p)

import torch

import test_norm_rotary_gpu as nr
import test_packed_attn_gpu as pa
import test_paged_attn_gpu as pg
from melspec_gpt_vqvae_amd import _ffi


def main():
    H = torch.float16
    assert _ffi.HALF_DTYPE == H and _ffi.LIB_PATH.endswith("libmelgpt_hip_fp16.so")
    for il in (False, True):
        nr.check_forward(65, 32, 8, 128, 128, il, H)
        nr.check_backward(65, 7, 1, 80, 32, il, H)
    nr.check_append(H, 16, 4, 64, 32, True, True, 16, [70, 1, 129], [0, 100, 63])
    print("norm and rotation ok", flush=True)
    for D in (64, 128):
        pa.check([64, 1, 63, 65, 200], [64, 1, 63, 65, 200], 4, 2, D, H)
        pa.check([5, 300, 129], [40, 301, 129], 4, 1, D, H)
        pa.check([70, 33, 3], [10, 0, 3], 4, 2, D, H)
    pa.test_values_that_are_not_finite_reach_only_the_queries_that_see_them(200, 128, "half")
    pa.test_few_queries_over_many_keys()
    print("packed attention ok", flush=True)
    pa.test_output_in_two_halves(64)
    pa.test_backward_with_few_key_heads(7, 1, 64)
    pg.check([300, 0, 128, 129, 1, 1100, 256], 7, 1, 128, 32, H, seed=3, extra_width=100)
    for D in (64, 128):
        pg.check([0, 1, 31, 129, 0, 500], 16, 2, D, 16, H)
        pa.test_output_in_two_halves(64)
    pa.test_backward_with_few_key_heads(7, 1, 64)
    pg.check([3000], 7, 1, D, 64, H)
    pg.test_prompt_then_tokens("half")
    print("all ok", flush=True)


if __name__ == "__main__":
    main()
