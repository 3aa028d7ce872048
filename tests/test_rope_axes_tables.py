"""Rotary tables of several axes are made where they are wanted.  No GPU."""
import pytest
import torch

from pom_b200.operators import precompute_freqs_axes


@pytest.mark.parametrize("device", [None, "cpu", "meta", torch.device("meta")])
def test_tables_on_a_device(device):
    got = precompute_freqs_axes((2, 3), (5, 7), device=device)
    want = precompute_freqs_axes((2, 3), (5, 7))
    for (c, s), (wc, ws) in zip(got, want):
        for a, b in ((c, wc), (s, ws)):
            assert a.device.type == torch.device(device or "cpu").type
            assert a.shape == b.shape and a.dtype == torch.float32
            if a.device.type == "cpu":
                assert torch.equal(a, b)
