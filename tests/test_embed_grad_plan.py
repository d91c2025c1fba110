"""How the embedding gradient is run, without a GPU: which problems it sorts, and that a problem whose
workspace is empty takes the one launch that uses none."""
import itertools

import pytest

import my_own_cnn_amd as M
from my_own_cnn_amd import _capi

TOKENS = [0, 1, 255, 256, 257, 682, 683, 1023, 1024, 1025, 8192, 8193, 10 ** 6, (1 << 31) - 65]
VOCABS = [1, 2, 1000, 1 << 20, (1 << 27) - 1, 1 << 27, (1 << 27) + 1, (1 << 28) - 1, 1 << 28]
CHANNELS = [1, 511, 512, 513, 1024, 1 << 20, 1 << 29]


def test_an_empty_workspace_and_no_sort_go_together():
    for vocab, c, tokens in itertools.product(VOCABS, CHANNELS, TOKENS):
        sorts, parts = M.plan_embed_grad(vocab, c, tokens)
        at = (vocab, c, tokens, sorts, parts)
        if M.embed_grad_workspace_size(vocab, c, tokens) == 0:
            assert (sorts, parts) == (0, 0), at
        else:
            assert tokens > 0 and sorts >= 1 and 1 <= parts <= tokens, at


def test_a_batch_without_tokens_is_never_sorted():
    for vocab, c in itertools.product(VOCABS, CHANNELS):
        assert M.plan_embed_grad(vocab, c, 0) == (0, 0), (vocab, c)
        assert M.embed_grad_workspace_size(vocab, c, 0) == 0


def test_sorts_by_tokens_channels_and_rows():
    assert M.plan_embed_grad(1000, 512, 1024)[0] == 0
    assert M.plan_embed_grad(1000, 512, 1025)[0] == 1
    assert M.plan_embed_grad(1000, 1024, 1024)[0] == 0  # 2048 workgroups
    assert M.plan_embed_grad(1000, 1025, 1024)[0] == 1
    assert M.plan_embed_grad(1000, 512, 8192)[0] == 1
    # keys 0 .. vocab in passes of up to 10 bits, two launches each
    for vocab, launches in [(1023, 2), (1024, 4), ((1 << 20) - 1, 4), (1 << 20, 6), (1 << 28, 6)]:
        assert M.plan_embed_grad(vocab, 512, 8193)[0] == launches, vocab
    # 256 tokens and fewer are not sorted for any table; more only up to 2^27 rows
    assert [M.plan_embed_grad(v, 1, 256)[0] for v in (1 << 27, (1 << 27) + 1, 1 << 28)] == [0, 0, 0]
    assert [M.plan_embed_grad(v, 1, 257)[0] for v in (1 << 27, (1 << 27) + 1, 1 << 28)] == [0, 1, 1]


def test_nothing_to_do_and_refusals():
    assert M.plan_embed_grad(0, 64, 9) == (0, 0) and M.plan_embed_grad(9, 0, 9) == (0, 0)
    with pytest.raises(M.MiqError, match=">= 0"):
        M.plan_embed_grad(-1, 64, 0)
    with pytest.raises(M.MiqError, match="2\\^28"):
        M.plan_embed_grad((1 << 28) + 1, 64, 0)
    assert M.lib().miq_plan_embed_grad(1, 1, 1, None) == _capi.MIQ_ERR_NULL_POINTER
