"""Importing the package builds no tensor and no autograd node, so it works in any mode and leaves
the GPU alone."""

import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
MODULES = ("visionhope_amd.models", "visionhope_amd.utils.causal_conv", "visionhope_amd.utils.state_space",
           "visionhope_amd.utils.gated_norm")


def _import(module, setup):
    code = f"import torch\n{setup}\n    import {module}\nassert not torch.cuda.is_initialized()\n"
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert run.returncode == 0, run.stderr


@pytest.mark.parametrize("module", MODULES)
def test_first_import_in_inference_mode(module):
    _import(module, "with torch.inference_mode():")


@pytest.mark.parametrize("module", MODULES)
def test_first_import_makes_no_tensor_on_the_default_device(module):
    """A tensor made at import would go to the default device, and could initialise the GPU."""
    _import(module, "torch.empty = torch.zeros = torch.ones = None\nwith torch.no_grad():")
