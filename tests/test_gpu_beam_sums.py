"""The sums of exponentials behind a selection, over long rows and many rows.

Logits alternate between 0 and -c, so that log sum exp is log(n / 2) + log(1 + e^-c).
An exponential is off by 2^-22 of itself at most and its argument's rounding (c
log2(e) <= 1: 2^-24 ln 2), the f32 sum of the 8 of a lane's chunk by 8 roundings,
what follows is 64 bits: below 2^-22 + 9 2^-24 = 8e-7 of the sum, together.  The scores
are f32's next to log sum exp, so that the candidates' sums come out small and exact.
"""
import numpy as np
import pytest

import static_lm as S

pytestmark = pytest.mark.gpu
TOL = 8e-7


def pick(torch, logits, scores, out):
    n = logits.shape[0]
    o = [torch.zeros(n, out, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]
    args = S.BeamSelectArgs(logits=logits.data_ptr(), ld=logits.stride(0), scores=scores.data_ptr(), num_groups=n, beams=1,
                            vocab=logits.shape[1], num_out=out, out_scores=o[0].data_ptr(), out_rows=o[1].data_ptr(),
                            out_tokens=o[2].data_ptr())
    size = S.beam_select_scratch_bytes(args)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    S.beam_select(args, scratch.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return [t.cpu().numpy() for t in o]


@pytest.mark.parametrize("rows,vocab,c", [(1, 1 << 30, 0.5), (1, 1 << 27, 0.5), (4800, 1 << 18, 0.25), (4, 1 << 18, 0.25)])
def test_sums_do_not_grow_worse_with_their_length(cuda, rows, vocab, c):
    """From one row cut into 128 parts to rows that are not cut, whose lanes take 128 chunks each."""
    logits = cuda.empty(rows, vocab, device="cuda")
    logits[:, 0::2] = 0
    logits[:, 1::2] = -c
    lse = np.log(vocab / 2) + np.log1p(np.exp(-c))
    scores = cuda.full((rows,), float(np.float32(lse)), device="cuda")
    got = pick(cuda, logits, scores, 2)
    want = float(np.float32(lse)) - lse
    assert (got[2] == [0, 2]).all() and (got[1] == np.arange(rows)[:, None]).all()
    assert np.abs(got[0] - want).max() <= TOL, np.abs(got[0] - want).max()
    del logits
    cuda.cuda.empty_cache()
