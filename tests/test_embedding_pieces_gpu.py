"""Rows that many tokens share, in a vocabulary split over ranks and in a whole one. Long runs of a row's tokens are summed in
blocks that begin anywhere among the sorted tokens of a call, so a piece may sum a row in another order than the whole table
does: each is held to the definition's bound, not to the other's bits."""
import pytest
import torch

import gpu_util
import indexed_util as iu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("tokens", [300, 1400])
def test_rows_of_many_tokens_in_pieces_and_in_the_whole_table(tokens, accumulate):
    import dfccl_amd
    gen = torch.Generator().manual_seed(tokens)
    rows, width, ranks, vocab = 10, 24, 3, 27  # the last piece is shorter
    grads = [torch.randn(tokens // 4 + 7 * r, width, generator=gen).to(gpu_util.DEVICE) for r in range(ranks)]
    ids = [torch.randint(0, vocab, (g.shape[0],), generator=gen) for g in grads]
    for i in ids:  # a frequent row in every piece, each some dozens to hundreds of tokens
        i[torch.rand(i.numel(), generator=gen) < 0.7] = 4
        i[torch.rand(i.numel(), generator=gen) < 0.4] = 15
        i[torch.rand(i.numel(), generator=gen) < 0.2] = 26
    ids = [i.to(gpu_util.DEVICE) for i in ids]
    old = torch.randn(vocab, width, generator=gen).to(gpu_util.DEVICE)
    pieces, whole = old.clone(), old.clone()
    for r in range(ranks):
        dfccl_amd.embedding_grad(grads, ids, pieces[r * rows:(r + 1) * rows], scale=0.5, first_row=r * rows, accumulate=accumulate)
    dfccl_amd.embedding_grad(grads, ids, whole, scale=0.5, accumulate=accumulate)
    torch.cuda.current_stream().synchronize()
    exact, before, count = iu.grad(grads, ids, vocab, 0, 0.5, None, old if accumulate else None)
    assert int((count > 16).sum()) >= 3
    iu.check(pieces, exact, before, "pieces")
    iu.check(whole, exact, before, "whole")
