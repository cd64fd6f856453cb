"""The 4-bit cache's decode where a group's scale decides: groups that are not numbers beside borders of units."""
import pytest
import torch

from oracle import kv4 as o4
from tests.test_gpu_kv4 import BF, DEV, HF, OPS, SCALE, _check_decode, _gen, _i64, _normal, _tables

pytestmark = pytest.mark.gpu


# ---- groups that are not numbers ------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("q_len,heads,kv_heads,lens", [
    (3, 8, 2, [65, 66, 130, 194]), (16, 1, 1, [65, 79, 70, 143]), (32, 1, 1, [65, 95, 128 + 20, 80]), (3, 14, 2, [65, 66, 130, 194]),
    (40, 2, 1, [70, 102, 134, 66]), (300, 1, 1, [330, 301, 364, 290])])
def test_groups_that_are_not_numbers_beside_a_border(q_len, heads, kv_heads, lens, dtype):
    """The newest tokens begin a unit (or half of one), so that in the one before, not seen whole by the first of them, the
    last see more tokens than it has. A value's group of scale 255 there makes NaN the group's dims, and no others."""
    g = _gen(21)
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    clean = pool.clone()
    bad = [(b, j, grp) for b, n in enumerate(lens) for j, grp in (((n - 1) // 64 * 64 - 60 + b, b), (5, (b + 2) % 4))]
    for b, j, grp in bad:
        pool[table[b, j // 128].long(), kv_heads - 1, o4.places(_i64([j % 128]))[3][0, grp]] = 255
    q = _normal(g, len(lens) * q_len, heads, 128, dtype=dtype)
    out, lse = OPS.kv4_decode(q, pool, table, _i64(lens), SCALE, q_len)
    nan = torch.zeros(len(lens), q_len, kv_heads, heads // kv_heads, 128, dtype=torch.bool, device=DEV)
    for b, j, grp in bad:
        first = max(0, j + q_len - lens[b])  # token t sees lens[b] - q_len + 1 + t keys
        nan[b, first:, -1, :, 32 * grp:32 * grp + 32] = True
    assert torch.equal(out.isnan(), nan.view(out.shape))
    want, _ = OPS.kv4_decode(q, clean, table, _i64(lens), SCALE, q_len)
    _check_decode(q, clean, table, lens, SCALE, q_len, (torch.where(nan.view(out.shape), want, out), lse))
