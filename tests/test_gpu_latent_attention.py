"""The example that runs the token operators together on the encoder graph's latents."""

import importlib.util
import pathlib

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("streams,frames,steps", [(2, 2, 16), (3, 5, 40), (1, 1, 1)])
def test_step_by_step_is_the_prompt(streams, frames, steps):
    path = pathlib.Path(__file__).resolve().parents[1] / "examples" / "latent_attention.py"
    spec = importlib.util.spec_from_file_location("latent_attention", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    r = example.run("codec_enc_tiny", streams, frames, steps)
    assert r["finite"]
    # The same queries on the same cached rows: both round the result to FP16
    # (2^-12 of it on average), the prompt its keys and values too (the step
    # scales them in FP32) and its weights: five such roundings in all.
    assert r["difference"] <= 5 * 2.0 ** -11, r
