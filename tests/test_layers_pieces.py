"""How the selective scan cuts a long prompt of few channels, without a GPU: the number of pieces from the size of the workspace."""
import importlib

import pytest

abi = importlib.import_module("burn-deltanet_b200._abi")
TILE, LEAST = 16, 128  # tokens between checkpoints, and of a piece at least


def pieces(seq, channels=1024, batch=1, state=16):
    a = abi.SelectiveScanArgs()
    a.batch, a.seq, a.channels, a.state, a.groups = batch, seq, channels, state, 1
    a.in_dtype = a.out_dtype = abi.DC_BF16
    floats = abi.lib().dc_selective_scan_workspace_size(a) // 4
    assert floats % (batch * channels) == 0
    return (floats // (batch * channels) + 1) // (state + 1)  # pieces * state end states and pieces - 1 sums of steps


@pytest.mark.parametrize("channels,batch,state", [(1024, 1, 16), (256, 2, 16), (64, 1, 4), (512, 1, 64), (2048, 1, 24)])
def test_three_or_more_pieces_or_none(channels, batch, state):
    for seq in (1, 127, 383, 384, 385, 400, 511, 512, 513, 700, 767, 768, 1000, 1023, 1024, 2047, 4096, 16384):
        n = pieces(seq, channels, batch, state)
        assert n == 0 or n >= 3, (seq, n)
        if n:
            longest = -(-(-(-seq // n)) // TILE) * TILE  # the shortest tiles' multiple that n pieces can share the tokens by
            assert longest >= LEAST - TILE and -(-seq // longest) == n, (seq, n)


def test_one_token_more_makes_no_longer_chain():
    """A piece's tokens grow with the prompt by whole tiles, not twofold at one length."""
    last = None
    for seq in range(384, 4096, 13):
        n = pieces(seq)
        piece = -(-(-(-seq // n)) // TILE) * TILE
        assert piece < 2 * LEAST + TILE and (last is None or piece <= last + 5 * TILE), (seq, n, piece)
        last = piece
