"""The workspace of attention: room for the parts of rows with many keys, whatever the offsets, and little more than that."""
import ctypes
import random

import pytest

F32, BF16 = 0, 1
A = 0x10000  # never dereferenced


def size(pkg, abi, back=0, **kw):
    p = pkg.Attention(A, A, A, 256, 64, 128, 64, 128, 64, A, A, 100, 200, 7, 4, 2, 64, 1, 1, 0, 0.125)
    for k, v in kw.items():
        setattr(p, k, v)
    return abi.dgs_attention_workspace_bytes(ctypes.byref(p), back)


def room(pkg, abi, **kw):
    """Parts that the workspace holds: 4 bytes of d + 2 values for each head of each."""
    more, less = (size(pkg, abi, heads=h, kv_heads=1, d=64, **kw) for h in (1024, 512))
    return (more - less) // (4 * 512 * 66)


def parts(q, k, tiles):
    """Of a sequence's rows (a part is 1 024 keys), if they are split at all."""
    if k <= 512 or q > 16 or (tiles and q >= 8 and k <= 4096):
        return 0
    return q * -(-k // 1024)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_room_for_all_parts(pkg, abi, dtype):
    rng = random.Random(1)
    keys = [0, 1, 512, 513, 514, 1023, 1024, 1025, 1026, 2048, 2049, 4096, 4097, 5120, 5121, 100_000]
    queries = [0, 1, 2, 7, 8, 9, 15, 16, 17, 300]
    sets = [[(q, k)] * n for q in queries for k in keys for n in (1, 2, 3, 50)]
    for _ in range(3000):
        some, few = rng.sample(keys, 2), rng.sample(queries, 2)
        sets.append([(rng.choice(few), rng.choice(some)) for _ in range(rng.choice([1, 2, 5, 40]))])
    for seqs in sets:
        n_q, n_k = sum(q for q, _ in seqs), sum(k for _, k in seqs)
        need = sum(parts(q, k, dtype != F32 and n_q >= 8) for q, k in seqs)
        for pad in (0, 1, 700):
            assert room(pkg, abi, n_q=n_q + pad, n_k=n_k + pad, seqs=len(seqs), dtype=dtype) >= need, (seqs[:4], len(seqs), pad)


def test_many_seeds_over_few_keys_each(pkg, abi):
    """A million seeds over ten million neighbours: less than K and V take (1 key head of 128, 16 bits), and less than the rows of q and out."""
    kw = dict(n_q=1_000_000, n_k=10_000_000, seqs=1_000_000, heads=16, kv_heads=1, d=128)
    assert size(pkg, abi, 0, **kw) < 1.8e9 and size(pkg, abi, 1, **kw) < 3.5e9
    assert size(pkg, abi, 1, **dict(kw, dtype=F32)) < 5.4e9
