"""Rules on logits whose lists are empty, or that name a list that is not there."""
import pytest
import torch

import ikv
from q8_ref import dev32

pytestmark = pytest.mark.gpu


def test_masks_of_no_rows_and_mask_of_without_masks_are_refused(dev):
    """Either would leave a row unrestricted that was to be held to a grammar."""
    x = torch.zeros(2, 40, device=dev)
    none = torch.empty(0, 2, dtype=torch.int32, device=dev)
    for bad in (dict(masks=none), dict(masks=none, mask_of=dev32([0, -1], dev)), dict(mask_of=dev32([0, -1], dev)),
                dict(mask_of=dev32([-1, -1], dev))):
        with pytest.raises(ValueError):
            ikv.adjust_logits(x, **bad)
