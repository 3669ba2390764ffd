"""l2c_decoder_beam_select's scores at the end of fp32's range: computed in 64 bits, rounded once."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_scores_below_the_lowest_number(torch_gpu, l2c):
    """Two continuations: the beam's score less nothing, and less 3e38. The second one's, -6e38, is finite in 64
    bits, so it is a continuation; stored it is -Inf, and on the next step its beam has none."""
    torch = torch_gpu
    beams, vocab = 3, 40
    logits = np.full((beams, vocab), -np.inf, np.float32)
    logits[:, 7], logits[:, 30] = 0.0, -3e38
    x = torch.from_numpy(logits).cuda()
    scores = torch.tensor([-3e38, -np.inf, -np.inf], device="cuda")
    tokens = torch.zeros(beams, dtype=torch.int32, device="cuda")
    parents = torch.zeros_like(tokens)
    ws = torch.empty(l2c.decoder_beam_workspace_bytes(vocab, beams, 1), dtype=torch.uint8, device="cuda")
    for _ in range(2):
        l2c.decoder_beam_select(scores, tokens, parents, None, x, scores, tokens, -1, vocab, beams, 1, 1, 0, ws)
        assert tokens.tolist() == [7, 30, -1] and parents.tolist() == [0, 0, -1]
        assert scores.tolist() == [float(np.float32(-3e38)), -np.inf, -np.inf]
