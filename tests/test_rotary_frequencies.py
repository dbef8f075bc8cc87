"""Defaults of torch_rbln_b200.rotary_frequencies."""

import torch


def test_the_fast_border_goes_by_the_scheme():
    """Turns from which a pair is left as it is: 4 for llama3, 32 for yarn, unless given."""
    from torch_rbln_b200 import rotary_frequencies as rf

    for scaling, high in (("llama3", 4.0), ("yarn", 32.0)):
        f, m = rf(128, 500000.0, scaling, 8.0, 8192)
        g, n = rf(128, 500000.0, scaling, 8.0, 8192, 1.0, high)
        assert torch.equal(f, g) and m == n
        assert not torch.equal(f, rf(128, 500000.0, scaling, 8.0, 8192, 1.0, 9.0)[0])
