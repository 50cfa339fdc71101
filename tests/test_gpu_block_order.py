"""Lists of many rows, four blocks of 16 keys to a tile, whose blocks come in any order, more than once, or not at all."""
import pytest
import torch

from test_gpu_block_attention import TYPES, check, make

pytestmark = pytest.mark.gpu

# Of some the last block is three behind the first, as if all four lay one behind the other.
TILES = [(0, 7, 5, 3), (5, 5, 5, 8), (0, 2, 1, 3), (0, 0, 0, 3), (2, 9, 1, 5), (2, -1, 9, 5), (4, 5, 99, 7), (6, 7, 8, 9), (12, 14, 13, 15), (3, 2, 1, 0),
         (9, 10, 10, 12), (1, 1, 3, 4)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("keys,heads,dim,causal", [(256, 8, 64, False), (256, 16, 128, True), (250, 8, 72, False), (320, 16, 40, True)])
def test_blocks_of_16_in_any_order(gpu, keys, heads, dim, causal, dtype):
    # 8 key-value heads times 4 batch entries times five blocks of queries: more than half a workgroup of 128 rows to a compute unit
    t = make(4, 320, keys, heads, 8, dim, TYPES[dtype], keys + dim)
    pos, crd = [0], []
    for row in range(160):
        tiles = [TILES[(row * 5 + i) % len(TILES)] for i in range(1 + row % 4)]
        crd += sum((list(x) for x in tiles), [])[:4 * len(tiles) - row % 7 % 4]
        pos.append(len(crd))
    pos, crd = (torch.tensor(x, dtype=torch.int32).cuda() for x in (pos, crd))
    check(gpu, "%s, %d keys, %d heads, dim %d, causal %s" % (dtype, keys, heads, dim, causal), t, pos, crd, 64, 16, causal)


def test_one_block_moved_in_every_tile(gpu):
    """Ascending lists give what they give in any other order of their blocks, each of them found by its own number."""
    t = make(4, 256, 256, 8, 8, 64, torch.bfloat16, 3)
    orders = [[0, 2, 1, 3], [3, 1, 2, 0], [1, 0, 3, 2], [0, 1, 2, 3]]
    crd = [4 * (x + row % 4) + i for row in range(128) for x in range(1 + row % 2) if x + row % 4 < 4 for i in orders[row % 4]]
    pos = [0]
    for row in range(128):
        pos.append(pos[-1] + 4 * sum(x + row % 4 < 4 for x in range(1 + row % 2)))
    check(gpu, "orders", t, *(torch.tensor(x, dtype=torch.int32).cuda() for x in (pos, crd)), 64, 16, True)
