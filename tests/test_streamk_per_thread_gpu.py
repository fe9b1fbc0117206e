"""Stream-K launches on the per-thread stream, which is one handle and another stream in every thread."""

import threading

import numpy as np
import pytest

from mlir_roller_amd import hip
from mlir_roller_amd.hip import DeviceArray, GemmConfig, GemmPlan, HipError
from oracle import gemm_oracle as go

pytestmark = pytest.mark.gpu
PER_THREAD = 2                                     # hipStreamPerThread


def test_the_librarys_workspace_serves_one_threads_stream(device):
    M, N, K = 1000, 1000, 1000
    plan = GemmPlan(GemmConfig(128, 128, 32, 64, 64, 16, 3, 0, 0, 4, 1, 3, 8, 0, 1, 0, 2))
    A, B = go.make_inputs(M, N, K, seed=5, distribution="integer")
    want = go.c_gemm_f32(A, B)
    dA, dB, dC, other = DeviceArray.from_host(A), DeviceArray.from_host(B), DeviceArray((M, N)), DeviceArray((M, N))
    plan.launch(dA, dB, dC, M, N, K, stream=PER_THREAD)
    plan.launch(dA, dB, dC, M, N, K, stream=PER_THREAD)
    ws = DeviceArray.zeros((plan.workspace_bytes(M, N, K)[0] // 4,), np.uint32)
    said = []

    def elsewhere():
        try:
            plan.launch(dA, dB, other, M, N, K, stream=PER_THREAD)
        except HipError as e:
            said.append(e)
        plan.launch(dA, dB, other, M, N, K, stream=PER_THREAD, workspace=ws)

    t = threading.Thread(target=elsewhere)
    t.start()
    t.join()
    hip.synchronize()
    assert len(said) == 1 and said[0].status == hip.RL_ERR_INVALID_ARG and "per-thread" in str(said[0])
    assert np.array_equal(dC.get(), want) and np.array_equal(other.get(), want)
