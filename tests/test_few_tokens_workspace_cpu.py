"""The workspace of the expert layer of a few tokens: what the layer takes asks for it, what it refuses asks for none."""
import pytest


def test_workspace_follows_the_pairs():
    from sglang_amd._lib import lib

    size = lib.sglamd_fused_experts_few_tokens_workspace
    for m in range(1, 66):
        for topk in range(1, 66):
            assert size(m, 16384, topk) == (m * topk * 16384 * 4 if m * topk <= 64 else 0), (m, topk)
    for m, i, topk in ((64, 16400, 1), (1, 16400, 1), (-1, 64, 2), (2, 64, -1), (2, -64, 2), (1 << 40, 64, 1), (1, 64, 1 << 20)):
        assert size(m, i, topk) == 0


@pytest.mark.parametrize("m,topk", [(13, 5), (64, 64), (65, 1), (1, 65)])
def test_more_pairs_are_refused_with_or_without_room_for_them(m, topk):
    from sglang_amd._lib import lib

    # x, xs, q_dtype, M, H, I, E, topk, w13, s13, b13, w2, s2, b2, weights, ids, ids_dtype, out, out_dtype, factor, ws, bytes, stream
    for room in (0, 1 << 40):
        args = [64, 64, 4, m, 256, 128, 8, topk, 64, 64, None, 64, 64, None, 64, 64, 5, 64, 2, 1.0, 64, room, None]
        assert lib.sglamd_fused_experts_few_tokens(*args) == -2
        assert b"pairs" in lib.sglamd_last_error()
