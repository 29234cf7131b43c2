"""Calls of the paged cache's operators that are refused, recorded or have to
leave something as it was, on the CPU (KILN_HIP_INTERPRET=1: the library's CPU
meaning)."""

import ctypes

import pytest
import torch

import kiln
import paged_reference as ref
from kiln.hip import lib as kl


@pytest.fixture(autouse=True)
def interpreting(monkeypatch):
    monkeypatch.setenv("KILN_HIP_INTERPRET", "1")


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


# -- the C entries -----------------------------------------------------------------------------


@pytest.mark.parametrize("stride", ["kp_t", "vp_t", "k_n", "v_n"])
def test_negative_token_strides_are_refused(stride):
    """The kernels count rows inside a tile with unsigned 32-bit offsets."""
    op = kl.Paged(kl.PAGED_ATTENTION, 1, 2, 1, 1, 64, 16, 4, 2, 0, kl.TYPE_F32, kl.TYPE_F32, 0, 1.0)
    size = ctypes.c_size_t()
    assert kl.load().kh_paged_workspace_bytes(op, size) == kl.OK
    setattr(op, stride, -64)
    assert kl.load().kh_paged_workspace_bytes(op, size) == kl.ERR_INVALID
    assert kl.load().kh_paged_host(op) == kl.ERR_INVALID
    assert b"negative" in kl.load().kh_last_error()
    launch = kl.LaunchDesc()
    launch.family, launch.variant, launch.n_refs, launch.rank = kl.FAM_PAGED, kl.PAGED_ATTENTION, 8, 6
    for i, x in enumerate((1, 2, 1, 1, 64, 16)):
        launch.shape[i] = x
    launch.gemm[0], launch.gemm[1] = 4, 2
    at = {"k_n": (1, 1), "v_n": (2, 1), "kp_t": (3, 2), "vp_t": (4, 2)}[stride]
    launch.refs[at[0]].strides[at[1]] = -64
    handle = ctypes.c_void_p()
    assert kl.load().kh_plan_create(ctypes.byref(launch), 1, ctypes.byref(handle)) == kl.ERR_INVALID
