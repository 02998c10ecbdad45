"""8-bit pages under tensor parallelism: a rank's shard of heads gives the bits that these heads have in the whole model."""
import dataclasses

import pytest
import torch

from agens_engine_b200.models import config as C
from agens_engine_b200.models.dense import DenseModel
from agens_engine_b200.ops import basic
from agens_engine_b200.ops import kv8 as K
from agens_engine_b200.parallel.tp_model import local_config

from tests.kv8_reference import FMTS
from tests.test_kv8_gpu import DEV, bf, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("world", [2, 4, 8])
def test_shards_store_attend_and_read_the_bits_of_the_whole(fmt, world):
    hq, hkv, hd = 64, 8, 128
    lens, new = [300, 1000, 17], [1, 5, 2]
    torch.manual_seed(world)
    n = max(lens)
    need = [(x + 15) // 16 for x in lens]
    bt = torch.full((3, max(need)), -1, dtype=torch.int32)
    order = torch.randperm(sum(need)).to(torch.int32)
    at = 0
    for s, m in enumerate(need):
        bt[s, :m] = order[at:at + m]
        at += m
    bt = bt.to(DEV)
    pos = i32([p for x in lens for p in range(x)])
    seq = i32([s for s, x in enumerate(lens) for _ in range(x)])
    rows = sum(lens)
    q_heads, k_heads, v_heads = (bf(torch.randn(rows, h, hd)).to(DEV) for h in (hq, hkv, hkv))
    inv = basic.rope_inv_freq(hd, 1e6, DEV)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    qr = [x - r + j for x, r in zip(lens, new) for j in range(r)]
    idx = (i32([0, 1, 6]), i32(new), i32(qr), i32([s for s, r in enumerate(new) for _ in range(r)]))
    last = torch.cat([torch.arange(sum(lens[:s + 1]) - r, sum(lens[:s + 1])) for s, r in enumerate(new)])

    def run(r, w):
        a, b = hq // w, hkv // w
        qkv = torch.cat([t[:, r * h:(r + 1) * h].reshape(rows, -1) for t, h in ((q_heads, a), (k_heads, b), (v_heads, b))], 1)
        pool = K.make_pool(sum(need), b, hd, DEV)
        q = torch.empty(rows, a * hd, dtype=torch.bfloat16, device=DEV)
        K.rope_kvstore8(qkv, a, b, hd, inv, pos, seq, bt, pool, fmt, q, status=st)
        out = K.attn_decode8(q[last.to(DEV)], pool, fmt, bt, *idx, a, b, hd, split_keys=128, status=st)
        return q.view(rows, a, hd), pool, out.view(-1, a, hd), K.kv_read8(pool, fmt, bt[1], n_tokens=n, status=st)

    whole = run(0, 1)
    for r in range(world):
        a, b = hq // world, hkv // world
        q, pool, out, read = run(r, world)
        hq_of, hkv_of = slice(r * a, (r + 1) * a), slice(r * b, (r + 1) * b)
        assert torch.equal(q, whole[0][:, hq_of]) and torch.equal(pool, whole[1][:, hkv_of])
        assert torch.equal(out, whole[2][:, hq_of]) and torch.equal(read, whole[3][:, :, hkv_of])
    assert int(st.item()) == 0


@pytest.mark.parametrize("world", [1, 2, 4, 8])
def test_a_shards_pool_split_and_bytes(world):
    cfg = dataclasses.replace(C.scaled(C.dense_32b(seed=0), 2), kv_cache="fp8")
    m = DenseModel(local_config(cfg, world), DEV, max_seqs=3, max_ctx=8192, n_pages=40)
    assert m.kv8 == "fp8" and all(t.shape == (40, 8 // world, 32 * 128 + 128) for t in m.kv)
    assert m.split8 == K.split_keys_for(8192, 3 * 8 // world)
    assert sum(t.numel() for t in m.kv) == 40 * 16 * cfg.kv_bytes_per_token(world)
    assert m.part8.numel() == K.part_floats(m.max_rows, 64 // world, 128, 8192, m.split8)
    assert m._stage.numel() * 2 == 8192 * (cfg.kv_dim // world) * 4
