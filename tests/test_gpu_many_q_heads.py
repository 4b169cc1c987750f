"""More q heads per KV head than a decode item holds (32): tiles, or a refusal; never rows left out."""

import numpy as np
import pytest

from tests.q4_scenario import D, Q4Scenario
from tests.scenario import Scenario
from yaxus_amd._lib import YxError

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,rows", [(33, 1), (40, 1), (40, 5), (128, 1), (128, 3)])
def test_a_4_bit_arena_takes_tiles(hip, hq, rows):
    sc = Q4Scenario(hip, 40, 16, 1, pool_seed=4)
    try:
        seqs = [sc.cache.new_seq() for _ in range(2)]
        sc.fill(dict(zip(seqs, [300, 17])))
        sc.begin([(s, rows) for s in seqs])
        k, v = sc.new_kv_rows()
        q = sc.draw(2 * rows, hq * D)
        got = hip.attend_append(sc.kv, 0, k, v, q, hq)
        sc.keep(k, v)
        sc.check(got, q, hq)
        hip.set_option("prefill_min_rows", 100)  # decode items asked for
        with pytest.raises(YxError, match="more than 32 query heads"):
            hip.attend(sc.kv, 0, q, hq)
    finally:
        hip.set_option("prefill_min_rows", 0)
        sc.kv.destroy()


def test_beyond_a_tile_it_refuses(hip):
    sc = Q4Scenario(hip, 8, 16, 1)
    try:
        sc.begin([(sc.cache.new_seq(), 1)])
        with pytest.raises(YxError, match="more query heads per KV head"):
            hip.attend(sc.kv, 0, np.zeros((1, 129 * D), np.float32), 129)
    finally:
        sc.kv.destroy()


@pytest.mark.parametrize("hq,rows", [(33, 1), (40, 1), (64, 3)])
def test_a_binary16_arena_refuses_them_in_decode_items(hip, hq, rows):
    sc = Scenario(hip, pages=40, page=16, hkv=1, pool_seed=4)
    try:
        seqs = [sc.cache.new_seq() for _ in range(2)]
        sc.run_pass([(s, 200) for s in seqs])
        sc.run_pass([(s, rows) for s in seqs])
        with pytest.raises(YxError, match="more than 32 query heads"):
            hip.attend(sc.kv, 0, np.zeros((2 * rows, hq * D), np.float32), hq)
    finally:
        sc.kv.destroy()
