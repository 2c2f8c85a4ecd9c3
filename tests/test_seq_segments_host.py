"""Which sequences of the delta rule's forward are walked in segments, seen without a GPU: segments
have states and maps in the workspace, everything else in it grows evenly with the chunks."""
import ctypes as C
import os

import pytest

import test_seq_host as H


@pytest.fixture(scope="module")
def segments():
    lib = C.CDLL(os.path.join(H.REPO, "tma-depthwise-conv_b200", "libtdc_sm100.so"))
    lib.tdc_delta_fwd_workspace.restype = C.c_int64

    def size(chunks, **o):
        return lib.tdc_delta_fwd_workspace(C.byref(H._delta(T=64 * chunks, dtype=H.CODES["TDC_BF16"], **o)))

    def count(chunks, B, HV, K, V):
        o, unit = dict(B=B, H=HV, HV=HV, K=K, V=V), B * HV * (K * V + K * K) * 4
        # (every part is a multiple of 256 bytes: the step of four chunks from sizes never split)
        step = (size(6, **o) - size(2, **o)) / 4
        extra = size(chunks, **o) - size(2, **o) - (chunks - 2) * step
        assert abs(extra - round(extra / unit) * unit) < unit / 8
        return max(1, round(extra / unit))

    return count


def test_short_sequences_are_walked_whole(segments):
    # joining 10 segments of 128 x 128 took longer than walking 13 chunks
    for chunks in range(2, 14):
        assert segments(chunks, 1, 4, 128, 128) == 1
    for chunks in range(2, 9):
        assert segments(chunks, 2, 4, 64, 64) == 1


def test_long_sequences_take_as_many_segments_as_pay(segments):
    assert 3 <= segments(40, 1, 4, 128, 128) <= 9
    assert segments(128, 1, 32, 128, 128) == 3           # as many as the SMs hold
    assert segments(40, 2, 4, 64, 64) >= 5
    for chunks in (2, 40, 500):
        assert segments(chunks, 8, 32, 128, 128) == 1    # enough walks without
