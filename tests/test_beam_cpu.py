"""Refusals of the beam search's kernels, checked where they are made: on the host, before any launch."""

from __future__ import annotations

import pytest
import torch

import beam_refusals
from mini_gpt_inference_b200.kernels import library
from mini_gpt_inference_b200.kernels.library import KernelLibraryError
from mini_gpt_inference_b200.kernels.ops import CudaOps


class NoLaunch:
    """The library's size functions, and no kernel."""

    def __getattr__(self, name):
        if name.endswith(("_floats", "_bytes")):
            return getattr(library.load(), name)
        raise AssertionError(f"{name} was reached")


@pytest.fixture()
def ops():
    ops = CudaOps.__new__(CudaOps)
    ops.device, ops.lib, ops.index, ops.launches = torch.device("cpu"), NoLaunch(), 0, 0
    return ops


def test_refusals(ops):
    names = []
    for name, call in beam_refusals.calls(ops, "cpu"):
        with pytest.raises(KernelLibraryError):
            call()
            pytest.fail(f"not refused: {name}")
        names.append(name)
    assert len(names) == len(set(names)) > 40
