"""Which kernel and cut the feed-forward block's products take at the tests' sizes: a change of the rule that chooses must
not leave a kernel's paths untested without a word."""
import pytest

from ltxattn import Failure, _lib, gated_ffn_plan
from test_gated_ffn_gpu import SIZES
from test_gated_ffn_paths_gpu import EXCHANGE, WIDE

PRODUCTS = ("inner", "out", "dinner", "dx")


@pytest.mark.parametrize("m,hidden,inner,out", WIDE)
def test_all_products_of_many_tokens_take_the_pairs_and_some_of_them_two_tiles(m, hidden, inner, out):
    assert gated_ffn_plan(m, hidden, inner, out) == dict.fromkeys(PRODUCTS, (1, 0, 0))
    tiles = lambda rows, cols, width=256: -(-rows // 256) * -(-cols // width)
    pairs = 74  # of 148 SMs
    assert tiles(m, inner, 128) > pairs and tiles(m, inner) > pairs and tiles(m, out) > pairs and tiles(m, hidden) > pairs
    assert 2 * tiles(inner, hidden) + tiles(out, inner) > 2 * pairs


@pytest.mark.parametrize("m,hidden,inner,out,columns,cluster", EXCHANGE)
def test_first_products_that_exchange_their_sums_in_two_pieces(m, hidden, inner, out, columns, cluster):
    # both accumulators' sums of 104 tokens fit beside each other
    assert gated_ffn_plan(m, hidden, inner, out)["inner"] == (2, columns, cluster)
    assert columns > 104


def test_every_product_takes_both_kernels_somewhere():
    plans = [gated_ffn_plan(*s[:4]) for s in SIZES + WIDE + EXCHANGE]
    for p in PRODUCTS:
        assert {plan[p][0] for plan in plans} == {1, 2}
    # and the CTAs that share a tile are one, some and as many as may be
    assert {plan[p][2] for plan in plans for p in PRODUCTS} >= {1, 2, 3, 4, 5, 6, 8}


def test_plans_without_tokens_and_refusals():
    assert gated_ffn_plan(0, 64, 128, 64) == dict.fromkeys(PRODUCTS, (0, 0, 0))
    for sizes in ((-1, 64, 64, 64), (1, 0, 64, 64), (1, 64, 60, 64)):
        with pytest.raises(Failure):
            gated_ffn_plan(*sizes)
    assert _lib.load().ltxattn_gated_ffn_plan(1, 64, 64, 64, None) == _lib.ERR_ARG
