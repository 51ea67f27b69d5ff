"""GPU: calls of packed_attention and KvPages that their documentation allows and that are easily got wrong. The oracle and its tolerance
are test_paged_gpu's."""
import pytest
import torch

from oracle_amd.paged import KvPages
from test_paged_gpu import attention64, close, filled, ints

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF, FP = torch.bfloat16, torch.float16


# Columns that see keys of an item and columns that end in front of it, in turn, where a NaN behind some limits makes the item run column by column: a
# column without keys must not disturb the one before it, whose parts are still being joined.
@pytest.mark.parametrize('n, hq, hkv', [(16, 1, 1), (8, 4, 2), (32, 2, 2), (64, 8, 2)])
@pytest.mark.parametrize('hd, dtype', [(128, BF), (64, FP)])
def test_attend_columns_without_keys_behind_columns_with_keys(n, hq, hkv, hd, dtype):
    prefix = 1024
    c, dense = filled(n, prefix, [i % 3 for i in range(n)], 64, hkv, hd, dtype, 80 + n)
    for token in (200, 500, 900):
        c.kv[1, 1, int(c.table[0, token // 64]), :, token % 64, 7] = float('nan')
    q, rows = torch.randn(n, hq, hd, device=DEV).to(dtype), ints(list(range(n)))
    for most in (180, 499, 899):                      # of each item: some columns end inside, every other one at once
        limits = [most - 37 * (i % 5) if i % 2 == 0 else (0, -1, 1)[i // 2 % 3] for i in range(n)]
        first = c.attend(1, q, rows, prefix_tokens=prefix, limits=ints(limits))
        for _ in range(30):
            assert torch.equal(c.attend(1, q, rows, prefix_tokens=prefix, limits=ints(limits)).nan_to_num(99.0), first.nan_to_num(99.0))
        c.check()
        for i, m in enumerate(limits):
            if m <= 0:
                assert (first[i] == 0).all()
            else:
                k, v = (x[:, :m] for x in dense[i])
                ref, tol = attention64(q[i], k, v, hd ** -0.5)
                keep = [d for d in range(hd) if d != 7 or m <= 200]       # `dense` was taken before the NaN went in
                close(first[i][:, keep], ref[:, keep], tol[:, keep], (most, i))
                assert 7 in keep or first[i, :, 7].isnan().all()
