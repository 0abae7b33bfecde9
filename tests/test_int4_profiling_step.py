"""A profiling run has no metadata: every way into a layer step gives zeros then."""

import pytest
import torch

from oscar_new_amd.backend import OscarAttentionImpl
from oscar_new_amd.config import OscarConfig


@pytest.mark.parametrize("bits", [2, 4])
def test_without_metadata(bits):
    impl = OscarAttentionImpl.standalone(6, 256, 1 / 16, 1, cfg=OscarConfig(history_bits=bits))
    q, k = torch.ones(3, 6, 256), torch.ones(3, 1, 256)
    for step in (impl.forward_appended(q, k, k, None, None, None, torch.ones(3, 1536)),
                 impl.forward(None, q, k, k, None, None, torch.ones(3, 1536))):
        assert step.shape == (3, 1536) and not bool(step.any())
    with pytest.raises(RuntimeError, match="no rotations"):
        impl.forward_appended(q, k, k, q, None, object(), torch.ones(3, 1536))
