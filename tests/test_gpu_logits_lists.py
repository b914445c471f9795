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


def test_lengths_past_an_empty_list_are_flagged(dev):
    x = torch.randn(3, 50, device=dev)
    none = torch.empty(3, 0, dtype=torch.int32, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    for lists in (dict(history=none, presence=torch.ones(3, device=dev)),
                  dict(bias_tokens=none, bias_values=none.float())):
        name = "n_history" if "history" in lists else "n_bias"
        for n, flag in (([0, 0, 0], 0), ([0, 1, 0], 1), ([-1, 0, 0], 1), ([0, 0, 2 ** 30], 1)):
            status.zero_()
            out = ikv.adjust_logits(x, **lists, **{name: dev32(n, dev)}, status=status)
            assert status.item() == flag and torch.equal(out, x)
