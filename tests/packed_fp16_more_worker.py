"""Child process of tests/test_packed_fp16_more_gpu.py (test infrastructure): checks of the packed-sequence operators on the
IEEE-half flavour of the library (MELGPT_HALF=fp16), at head sizes and heads beside those of packed_fp16_worker."""
import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
for p in (os.path.dirname(HERE), HERE):
    sys.path.insert(0, p)

import torch

import packed_norms as N
import test_packed_attn_gpu as pa
import test_packed_edges_gpu as pe
import test_packed_norms_gpu as pn
import test_paged_attn_gpu as pg
from melspec_gpt_vqvae_amd import _ffi


def main():
    H = torch.float16
    assert _ffi.HALF_DTYPE == H and _ffi.LIB_PATH.endswith("libmelgpt_hip_fp16.so")
    for D in (64, 128):
        pa.test_output_in_two_halves(D)
        pe.test_output_and_its_remainder_fit_each_other(D)
        pg.check([3000], 7, 1, D, 64, H)
        print("two halves, 3000 cached keys", D, "ok", flush=True)
    for heads in ((7, 1, 64), (8, 2, 128), (5, 1, 128)):
        pa.test_backward_with_few_key_heads(*heads)
        print("few key heads", heads, "ok", flush=True)
    for i, case in enumerate(N.CASES):
        pn.check(*case, H, i)
    print("norms ok", flush=True)
    for il in (False, True):
        pe.test_values_beyond_the_rotation_pass_unchanged(5, 3, 2, 64, 32, il, "half")
    pe.test_log_sums_of_rows_that_no_sequence_owns([4, 20], [50, 2080], "half")
    for D in (64, 128):
        pe.test_one_long_sequence_in_a_packed_batch(D, 31)
    pe.test_long_sequences_in_a_large_batch_of_short_ones(16, 8, 64, "half")
    print("all ok", flush=True)


if __name__ == "__main__":
    main()
