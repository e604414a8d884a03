"""Chunks of causal_conv's gradients, by the size of their workspace, on the host: no GPU is touched."""
import pytest

from m2_b200 import _lib


@pytest.mark.parametrize("batch,length,dim,taps,chunks", [
    (3, 2048, 1536, 4, 49),      # bf16, 4 channels a thread, 3 blocks of 128 threads on each of 148 multiprocessors: 56832 threads for 3 x 384; float32 has 24
    (3, 2048, 1536, 8, 32),      # 2 blocks an SM with more than 4 taps: 37888 threads
    (16, 2048, 1536, 4, 9),
    (16, 2048, 1536, 8, 12),     # 6 in one round are 342 tokens: two rounds of 171 (float32: 4 in one, two rounds of 256)
    (64, 8192, 1536, 4, 32),     # 256 tokens at most
    (1, 100, 8, 4, 7)])          # 16 at least
def test_chunks_are_whole_rounds_of_the_threads_that_run_at_once(batch, length, dim, taps, chunks):
    assert _lib.lib().m2_causal_conv_workspace(batch, length, dim, taps) == 4 * batch * chunks * (taps + 1) * dim
