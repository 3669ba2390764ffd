"""l2c_decoder_logprobs against its formulas by a bound for what a lane adds in fp32: 16 exponentials at most, 15 roundings,
2^-20 of the sum; 2^-22 for an exponential, and a distance t from the largest logit rounded before it, t 2^-24 of it, which
d, the mean of t by the probabilities, says of the sum. The entropy has d's sums beside log Z, whose terms are t times as
large: the mean of t^2 takes the place of d there."""
import pytest
import torch
from test_logprobs_gpu import close, want_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab,spread", [(1, 16, 1.0), (3, 1024, 3.0), (2, 32000, 3.0), (600, 4099, 1.0), (520, 9001, 8.0),
                                               (1, 131072, 0.01)])
def test_sums_of_sixteen(torch_gpu, l2c, rows, vocab, spread):
    print(f"case bounds {rows}x{vocab} {spread}", flush=True)
    gen = torch.Generator("cuda").manual_seed(vocab)
    x = spread * torch.randn(rows, vocab, generator=gen, device="cuda")
    tokens = torch.randint(vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    workspace = torch.empty(l2c.decoder_logprobs_workspace_bytes(vocab, 4, rows), device="cuda", dtype=torch.uint8)
    logprobs, entropies = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    top_tokens = torch.empty(rows, 4, device="cuda", dtype=torch.int32)
    top_logprobs = torch.empty(rows, 4, device="cuda")
    l2c.decoder_logprobs(logprobs, entropies, top_tokens, top_logprobs, x, tokens, vocab, 4, rows, workspace)
    mine, entropy, which, alternatives, d = want_of(x, tokens, 4)
    y = x.double() - x.double().amax(1, keepdim=True)
    square = (torch.softmax(y, 1) * y * y).sum(1)
    e = 2.0 ** -20 + 2.0 ** -22
    off = e + d * 2.0 ** -24  # of log Z
    assert torch.equal(top_tokens.long(), which)
    close(logprobs, mine, off)
    close(top_logprobs, alternatives, off.unsqueeze(1).expand(rows, 4))
    close(entropies, entropy, off + 2 * e * d + (d * d + square) * 2.0 ** -24)
