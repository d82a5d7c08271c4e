"""The timeline variant stamps the kernels with an epilogue too, into the variables that are read back."""
import numpy as np
import pytest


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ("none", "gelu_tanh"))
@pytest.mark.parametrize("M,N,K", [(512, 512, 512), (4096, 4096, 1024)])
def test_stamps_of_the_epilogue_are_in_program_order(M, N, K, activation):
    from rocm_wmma_gemm_b200 import timeline
    r = timeline.run(timeline.load(), "bf16_bf16", M, N, K, launches=8, activation=activation)
    c = r["cycles_after_wait"]
    # entry, set-up, wait (= 0), first / last TMA, first full, last commit, drained, seen, first / last store, read, tail, freed
    assert np.isfinite(c).all()
    assert c[0] < c[1] and c[2] == 0
    assert 0 < c[3] < c[5] < c[6] and c[3] <= c[4] and c[6] <= c[7]
    assert c[5] < c[8] < c[9] <= c[10] < c[11] < c[13] and c[6] < c[10]
    t = r["cta_times"]
    live = t[1] > 0
    assert live.any() and np.all(t[0][live] <= t[2][live]) and np.all(t[2][live] <= t[1][live])
