"""Memory that a backward pass of jagged_attention asks for, from the C entry alone; the planes of its statistics."""
import ctypes

import pytest


def _size(pdm, seqs, tokens, window, sinks, hk=8, group=1, D=128):
    L = pdm._lib
    d = L.JaggedAttentionDesc(L.PDM_BF16, hk * group, hk, D, seqs, 1, window, sinks, 0, 0, 0.125, 0, tokens, tokens, hk * group * D, D,
                              hk * D, D, hk * D, D)
    return L.lib().pdm_jagged_attention_bwd_workspace_size(ctypes.byref(d), 0)


@pytest.mark.parametrize("seqs,length,window,sinks", [(16_384, 100, 1_024, 4), (65_536, 100, 1_024, 4), (4_096, 300, 1_024, 512),
                                                      (512, 300, 1_024, 1_024), (100_000, 20, 64, 4)])
def test_sinks_of_short_sequences(pdm, seqs, length, window, sinks):
    """None of them is longer than the window.  Sums are kept for the sinks of as many sequences as could be: sinks rows, in fp32, for
    dk and dv and twice over, of window + 1 tokens."""
    without, extra = _size(pdm, seqs, seqs * length, window, 0), 2 * 2 * 4 * 8 * 128
    bound = without + seqs * length // (window + 1) * min(sinks, window + 1) * extra
    assert 0 < _size(pdm, seqs, seqs * length, window, sinks) <= bound
    assert sinks > 4 or window < 1_024 or bound < 2 ** 30


def test_sinks_of_few_sequences(pdm):
    """Sums for each sequence's sinks, times the shares of its queries, of which there are at most 1,024 for all heads."""
    for seqs, length, window, sinks in ((1, 100_000, 16, 4), (2, 8_000, 512, 4), (8, 2_000, 100, 1_024)):
        without, row = _size(pdm, seqs, seqs * length, window, 0), 2 * 4 * 8 * 128
        assert _size(pdm, seqs, seqs * length, window, sinks) <= without + seqs * sinks * row * (1024 // (8 * seqs) + 2)


def test_no_more_than_for_every_token(pdm):
    for seqs, tokens, window, sinks in ((1_000, 100_000, 1, 1_024), (10, 100_000, 7, 1_024), (5_000, 5_000, 3, 9)):
        assert _size(pdm, seqs, tokens, window, sinks) <= _size(pdm, seqs, tokens, window, 0) + tokens * 2 * 2 * 4 * 8 * 128


def test_planes_of_the_statistics(pdm):
    L = pdm._lib
    for planes in (-1, 0, 1, 2, 3):
        d = L.JaggedAttentionDesc(L.PDM_BF16, 2, 1, 64, 1, 1, 0, 0, 0, 4, 0.125, planes, 8, 8, 128, 64, 64, 64, 64, 64)
        size = L.lib().pdm_jagged_attention_bwd_workspace_size(ctypes.byref(d), 1)
        assert size > 0 if 0 <= planes <= 2 else size == L.PDM_ERR_INVALID and "stats_planes" in L.last_error()
    p = 1 << 20  # never read
    d = L.JaggedAttentionDesc(L.PDM_BF16, 2, 1, 64, 1, 1, 0, 0, 0, 4, 0.125, 2, 8, 8, 128, 64, 64, 64, 64, 64)
    assert L.lib().pdm_jagged_attention_fwd(ctypes.byref(d), p, p, p, p, p, p, p, p, None, None, None, 0, None, None) == L.PDM_ERR_INVALID
    assert "out_rest without stats" in L.last_error()
