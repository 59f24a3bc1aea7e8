"""A batch is cleared before it is handed out: a prompt that is put in at once
stays."""
import numpy as np
import pytest

from huggingfaceeacp_amd import gemma_q8 as G
from test_gpu_decoder import build_pair
from gpu_helpers import seeded_weights, small_heads_shape

pytestmark = pytest.mark.gpu


def test_a_prompt_right_after_create_stays(torch_cuda):
    shape = small_heads_shape(max_positions=64)
    decoder, _ = build_pair(shape, seeded_weights(shape))
    rng = np.random.default_rng(11)
    for _ in range(20):
        batch = G.Batch(decoder, 5)
        prompts = [rng.integers(1, shape.vocab, n).astype(np.int32) for n in (3, 7, 1, 12, 20)]
        for s, prompt in enumerate(prompts):
            batch.prefill(s, prompt)
        for s, prompt in enumerate(prompts):
            assert list(batch.tokens(s, 0, len(prompt))) == list(prompt)
        batch.close()
