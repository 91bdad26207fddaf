"""Stricter forms of ``ffn_reference``'s comparison, and the sizes that reach every variant of the dense gated FFN's
tiled kernel."""

import torch

import ffn_reference as ref

_close = ref.close


def close(got, want, err):
    """``ffn_reference.close`` (which a NaN passes, being larger than no bound) on finite numbers only."""
    assert torch.isfinite(want).all() and torch.isfinite(err).all(), "the reference and its bounds are numbers"
    bad = int((~torch.isfinite(got)).sum())
    assert not bad, f"{bad} of {got.numel()} values are no numbers"
    assert got.shape == want.shape
    _close(got, want, err)


def even(got, want, roundings=3):
    """Every block of 64 x 64 outputs is off, in the root of its mean square, by less than `roundings` half steps.  A
    chain of roundings (an operand to 16 bits, the result, a residual's sum before it) whose signs are independent of the
    numbers adds at most a half step each; the bound on each output's sum grows with K and with the sum of magnitudes,
    and lets pass a stage of K that a long sum lacks, which a block's mean square does not: 64 of 16384 terms are 6 %
    of it, three half steps 1.2 % in bf16.  A block of small outputs is held to the whole result's mean square."""
    def blocks(t):
        r, c = (-t.shape[0]) % 64, (-t.shape[1]) % 64
        t = torch.nn.functional.pad(t, (0, c, 0, r))
        return t.reshape(t.shape[0] // 64, 64, t.shape[1] // 64, 64).sum((1, 3))

    size = blocks(torch.ones_like(want))
    scale = torch.maximum(blocks(want ** 2), size * (want ** 2).mean()).sqrt()
    off = blocks((got.double() - want) ** 2).sqrt() / scale
    assert float(off.max()) <= roundings * ref.HALF_STEP[got.dtype], (float(off.max()), ref.HALF_STEP[got.dtype])


# Training steps (tokens, d_model, d_ff) whose products, between them, take output tiles of 256 with every epilogue
# and operand layout, whole and in shares of K, with and without a rest of K (tests/test_gated_plan.py holds them to it)
STEPS = [(16384, 1024, 4096), (3001, 4104, 8200), (9537, 136, 3536), (154, 2112, 14912), (4161, 136, 3648), (161, 4160, 3816),
         (6953, 144, 2080), (7885, 4376, 136), (64, 8856, 472), (64, 1080, 7520)]
