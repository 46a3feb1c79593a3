"""What the wrappers of the operators around the state path make of tensors' types, without a GPU."""
import pytest
import torch

import ssd_amd as ops
from test_layer_cpu import scan_args, step_args


def test_types_that_would_have_to_lose_bits_are_refused():
    x, w = torch.zeros(2, 8, 16), torch.zeros(16, 4)
    wrong = [lambda: ops._norm_fwd(x, torch.zeros(16), residual=x.double()), lambda: ops._norm_fwd(x.half(), torch.zeros(16), z=x.double()),
             lambda: ops._norm_fwd(x, torch.zeros(16), residual=x.int()),
             lambda: ops._short_conv_fwd(x, w, initial_states=torch.zeros(2, 16, 3, dtype=torch.float64))]
    for key in ("B", "C", "z"):
        wrong.append(lambda key=key: ops._ssd_scan_fwd(**{**scan_args(), key: scan_args()["x" if key == "z" else key].double()}))
        wrong.append(lambda key=key: ops._ssd_scan_step(**{**step_args(), key: step_args()["x" if key == "z" else key].double()}))
    for i, call in enumerate(wrong):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was taken")


def test_slots_and_lengths_are_whole_numbers():
    x, w = torch.zeros(2, 8, 16), torch.zeros(16, 4)
    for call in (lambda: ops._short_conv_fwd(x, w, lengths=torch.zeros(2)), lambda: ops._ssd_scan_fwd(**scan_args(), lengths=torch.zeros(1).half()),
                 lambda: ops._short_conv_step(x[:, 0], torch.zeros(3, 16, 3), w, slots=torch.zeros(2)), lambda: ops._ssd_scan_step(**step_args(), slots=torch.zeros(2))):
        with pytest.raises(AssertionError):
            call()
