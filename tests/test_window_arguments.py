"""Windows and first keys as whole numbers of any kind."""
import numpy as np
import pytest
import torch

import pypto_amd
from tests.test_prompt_refusals import attention, refused
from tests.test_serving_refusals import latent


@pytest.mark.parametrize("kind", [np.int64, np.int32, np.uint8])
def test_windows_of_numpy_s_whole_numbers(kind):
    for window, sinks in ((kind(5), 2), (5, kind(2)), (kind(5), kind(0))):
        refused(RuntimeError, "GPU", pypto_amd.latent_attention, latent(), window=window, sinks=sinks)
        refused(RuntimeError, "GPU", pypto_amd.prompt_window_attention, attention() + [window], sinks=sinks)
    refused(ValueError, "window", pypto_amd.latent_attention, latent(), window=kind(0))
    for bad in (np.float32(5), np.bool_(True), np.array([5]), torch.tensor(5), "5"):
        refused(ValueError, "window", pypto_amd.latent_attention, latent(), window=bad)
        refused(ValueError, "window", pypto_amd.prompt_window_attention, attention() + [bad])
        refused(ValueError, "sinks", pypto_amd.latent_attention, latent(), window=5, sinks=bad)
