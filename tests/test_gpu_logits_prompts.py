"""Which tokens of a row's text count as generated: those of the history from prompt_lens[s] on, and every draft before the
row, also where prompt_lens[s] is the history's length or passes it."""
import numpy as np
import pytest

from test_gpu_logits import run
from test_gpu_serving import F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prompt", [0, 3, 5, 6, 7, 4000000000])
@pytest.mark.parametrize("masked", [False, True])
def test_drafts_are_never_of_the_prompt(native, prompt, masked):
    vocab, rows = 40, 4
    history = np.array([[1, 2, 3, 2, 4, 30, 31]], np.uint32)     # five of them are text
    drafts = np.array([[1, 6, 6]], np.uint32)
    x = np.linspace(-3, 4, rows * vocab).astype(np.float32).reshape(1, rows, vocab)
    rep, freq, pres = (np.array([v], np.float32) for v in (1.5, 0.25, 0.5))
    mask = np.full((1, rows, 2), 0xFFFFFFFF, np.uint32) if masked else None
    got, _ = run(native, x, F32, 0, 0, True, vocab, history, np.array([5], np.uint32), np.array([prompt], np.uint32), drafts,
                 np.array([3], np.uint32), rep, freq, pres, None, None, None, mask)
    for t in range(rows):
        before = [int(v) for v in drafts[0, :t]]
        generated = [1, 2, 3, 2, 4][min(prompt, 5):] + before
        for v in range(vocab):
            want = x[0, t, v]
            if v in [1, 2, 3, 4] + before:
                want = want / rep[0] if want > 0 else want * rep[0]
            if v in generated:
                want = (want - freq[0] * np.float32(generated.count(v))) - pres[0]
            assert got[0, t, v] == want, (t, v)
