"""What the 8-bit key-value cache refuses, and its reference's own format, without a GPU."""
import ctypes as C

import pytest
import torch

from agens_engine_b200 import _lib
from agens_engine_b200.ops import kv8 as K

from tests.kv8_reference import FMTS, Cache, encode, fields, values

HQ, HKV, HD = 4, 2, 64


def _store_args(n=3):
    return dict(qkv=torch.zeros(n, (HQ + 2 * HKV) * HD, dtype=torch.bfloat16), hq=HQ, hkv=HKV, hd=HD, inv_freq=torch.zeros(HD // 2),
                tok_pos=torch.zeros(n, dtype=torch.int32), tok_seq=torch.zeros(n, dtype=torch.int32), block_table=torch.zeros(1, 4, dtype=torch.int32),
                pool=K.make_pool(4, HKV, HD, "cpu"), fmt="int8", q_out=torch.zeros(n, HQ * HD, dtype=torch.bfloat16))


def _attn_args(n=3):
    i = lambda m: torch.zeros(m, dtype=torch.int32)
    return dict(q=torch.zeros(n, HQ * HD, dtype=torch.bfloat16), pool=K.make_pool(4, HKV, HD, "cpu"), fmt="fp8", block_table=i(4).view(1, 4), grp_tok0=i(1),
                grp_cnt=i(1), tok_pos=i(n), tok_seq=i(n), hq=HQ, hkv=HKV, hd=HD)


BAD_STORE = [
    (dict(fmt="int4"), "format"), (dict(fmt=8), "format"), (dict(hkv=4), "KV heads"), (dict(hd=128), "KV heads"), (dict(hq=5), "qkv"),
    (dict(pool=torch.zeros(4, HKV, 100, dtype=torch.uint8)), "pages"), (dict(pool=torch.zeros(4, HKV, 2176, dtype=torch.int8)), "uint8"),
    (dict(pool=torch.zeros(4, 2 * HKV, 2176, dtype=torch.uint8)[:, ::2]), "contiguous"), (dict(pool=torch.zeros(0, HKV, 2176, dtype=torch.uint8)), "pages"),
    (dict(qkv=torch.zeros(3, 8 * HD)), "qkv"), (dict(qkv=torch.zeros(3, 16 * HD, dtype=torch.bfloat16)[:, ::2]), "unit stride"),
    (dict(qkv=torch.zeros(3, 8 * HD + 4, dtype=torch.bfloat16)[:, :8 * HD]), "boundaries"), (dict(qkv=torch.zeros(3, 8 * HD + 8, dtype=torch.bfloat16)[:, 1:8 * HD + 1]), "boundaries"),
    (dict(q_out=torch.zeros(2, HQ * HD, dtype=torch.bfloat16)), "q_out"), (dict(tok_pos=torch.zeros(3, dtype=torch.int64)), "tok_pos"),
    (dict(tok_seq=torch.zeros(2, dtype=torch.int32)), "tok_seq"), (dict(tok_pos=torch.zeros(6, dtype=torch.int32)[::2]), "tok_pos"),
    (dict(block_table=torch.zeros(4, dtype=torch.int32)), "block_table"), (dict(block_table=torch.zeros(4, 2, dtype=torch.int32).t()), "block_table"),
    (dict(block_table=torch.zeros(2, 0, dtype=torch.int32)), "block_table"), (dict(inv_freq=torch.zeros(HD)), "inv_freq"), (dict(inv_freq=torch.zeros(HD // 2).double()), "inv_freq"),
    (dict(rope_pos3=torch.zeros(3, 3, dtype=torch.int32)), "pair_axis"),
    (dict(rope_pos3=torch.zeros(2, 3, dtype=torch.int32), pair_axis=torch.zeros(HD // 2, dtype=torch.uint8)), "rope_pos3"),
    (dict(rope_pos3=torch.zeros(3, 3, dtype=torch.int32), pair_axis=torch.zeros(HD // 2, dtype=torch.uint8), rope_pos=torch.zeros(3, dtype=torch.int32)), "without rope_pos"),
    (dict(status=torch.zeros(1)), "status"), (dict(), "CUDA device"),
]


@pytest.mark.parametrize("change,word", BAD_STORE)
def test_store_refuses(change, word):
    with pytest.raises(ValueError, match=word):
        K.rope_kvstore8(**{**_store_args(), **change})


BAD_ATTN = [
    (dict(fmt="bf16"), "format"), (dict(hq=3), "multiple"), (dict(hkv=1, hq=4), "KV heads"), (dict(q=torch.zeros(3, HQ * HD, dtype=torch.float16)), "q:"),
    (dict(q=torch.zeros(3, HQ * HD + 4, dtype=torch.bfloat16)[:, :HQ * HD]), "boundaries"), (dict(out=torch.zeros(3, HQ * HD)), "out"),
    (dict(out=torch.zeros(2, HQ * HD, dtype=torch.bfloat16)), "out"), (dict(grp_cnt=torch.zeros(0, dtype=torch.int32)), "grp_cnt"),
    (dict(tok_pos=torch.zeros(2, dtype=torch.int32)), "tok_pos"), (dict(tree_mask=torch.zeros(3, dtype=torch.int64)), "tree_mask"),
    (dict(tree_mask=torch.zeros(2, dtype=torch.int32)), "tree_mask"), (dict(block_table=torch.zeros(1, 4)), "block_table"),
    (dict(split_keys=40), "split_keys"), (dict(split_keys=4096), "split_keys"), (dict(split_keys=0), "split_keys"), (dict(max_ctx=65), "max_ctx"), (dict(max_ctx=0), "max_ctx"),
    (dict(split_keys=16, part=torch.zeros(3 * HQ * 4 * (HD + 2) - 1)), "part"), (dict(part=torch.zeros(9999, dtype=torch.float64)), "part"),
    (dict(split_keys=16, part=torch.zeros(3 * HQ * 4 * (HD + 2))), "CUDA device"), (dict(), "CUDA device"),
]


@pytest.mark.parametrize("change,word", BAD_ATTN)
def test_attention_refuses(change, word):
    with pytest.raises(ValueError, match=word):
        K.attn_decode8(**{**_attn_args(), **change})


def test_read_refuses():
    pool, pages = K.make_pool(4, HKV, HD, "cpu"), torch.zeros(2, dtype=torch.int32)
    for kw, word in ((dict(n_tokens=33), "n_tokens"), (dict(n_tokens=-1), "n_tokens"), (dict(out=torch.zeros(2, 2, HKV, 16, HD)), "out"),
                     (dict(out=torch.zeros(1, 2, HKV, 16, HD, dtype=torch.bfloat16)), "out"), (dict(), "CUDA device")):
        with pytest.raises(ValueError, match=word):
            K.kv_read8(pool, "int8", pages, **kw)
    with pytest.raises(ValueError, match="pages"):
        K.kv_read8(pool, "int8", pages.long())
    with pytest.raises(ValueError, match="head_dim"):
        K.make_pool(4, 2, 96, "cpu")


def test_the_library_refuses_what_the_launchers_would_not_pass_on():
    """The C entries check their own arguments: nothing is launched (1 is a bad argument)."""
    lib = _lib.cuda_lib()
    s = _lib.Kv8StoreArgs(n=1, hq=1, hkv=1, n_seq=1, bt_cols=1, n_pages=1)
    for hd, fmt, kw in ((96, 0, {}), (64, 2, {}), (64, 0, dict(n=0)), (64, 0, dict(ld=4)), (128, 1, dict(n_pages=0)), (64, 0, dict(n_seq=0))):
        b = _lib.Kv8StoreArgs(n=1, hq=1, hkv=1, n_seq=1, bt_cols=1, n_pages=1)
        for k, v in kw.items():
            setattr(b, k, v)
        assert lib.b2_kv8_store(C.byref(b), hd, fmt, None) == 1
    for hd, fmt, kw in ((32, 0, {}), (64, -1, {}), (64, 0, dict(hq=3, hkv=2)), (64, 0, dict(n_groups=0)), (64, 0, dict(ldq=4)), (64, 0, dict(bt_cols=0)),
                        (64, 0, dict(split_keys=24)), (64, 0, dict(split_keys=4096)), (64, 0, dict(max_splits=0)), (64, 0, dict(max_splits=2)),
                        (64, 0, dict(n_tok=2 ** 31 - 1)), (64, 0, dict(n_groups=2 ** 26))):
        b = _lib.Kv8AttnArgs(n_pages=1, bt_cols=1, n_seq=1, n_groups=1, n_tok=1, hq=1, hkv=1, split_keys=256, max_splits=1)
        for k, v in kw.items():
            setattr(b, k, v)
        assert lib.b2_kv8_attn(C.byref(b), hd, fmt, None) == 1
    for bad in ((0, 1, 64, 0, 1, 0), (1, 0, 64, 0, 1, 0), (1, 1, 80, 0, 1, 0), (1, 1, 64, 5, 1, 0), (1, 1, 64, 0, 0, 0), (1, 1, 64, 0, 1, -1)):
        n_pages, hkv, hd, fmt, n_out, n_tok = bad
        assert lib.b2_kv8_read(_lib.packer(_lib.Kv8ReadArgs)(0, n_pages, hkv, 0, n_out, n_tok, 0, 0), hd, fmt, None) == 1


@pytest.mark.parametrize("cls", [_lib.Kv8StoreArgs, _lib.Kv8AttnArgs, _lib.Kv8ReadArgs])
def test_packed_arguments_are_the_structures_bytes(cls):
    values = [1000 + 7 * i if t is not C.c_float else 0.375 for i, (_, t) in enumerate(cls._fields_)]
    got = cls.from_buffer_copy(_lib.packer(cls)(*values))
    assert [getattr(got, name) for name, _ in cls._fields_] == values


def test_splits_for_a_context():
    sizes = (1, 700, 7040, 7041, 8000, 16000, 28160, 28161, 131072, 196608, 196609, 262145, 1 << 20)
    assert [K.split_keys_for(n) for n in sizes] == [128, 128, 128, 256, 256, 512, 512, 768, 768, 768, 1024, 2048, 2048]
    assert [K.split_keys_for(4000, h) for h in (2, 8, 16, 55, 56, 1000)] == [128, 128, 256, 512, 768, 768]
    assert [K.split_keys_for(n, 1) for n in (50000, 131072, 131073, 300000)] == [256, 512, 768, 2048]
    assert all(K.split_keys_for(n, h) % 16 == 0 and K.split_keys_for(n, h) <= K.MAX_SPLIT for n in range(1, 10 ** 6, 7919) for h in (1, 8, 512))
    assert K.part_floats(3, 8, 128, 256, 256) == 0 and K.part_floats(3, 8, 128, 257, 256) == 3 * 8 * 2 * 130 and K.part_floats(1, 2, 64, 100, 16) == 2 * 7 * 66


@pytest.mark.parametrize("fmt", FMTS)
def test_the_format_holds_rows_to_half_a_step(fmt):
    x = torch.randn(50, 2, HD) * torch.exp(3 * torch.randn(50, 1, 1))
    c = Cache([50], 2, HD, fmt, k=[x], v=[x])
    k, v = c.rows(0)
    scale = encode(x, fmt)[1].double().unsqueeze(-1)
    step = 0.5 * scale if fmt == "int8" else 2.0 ** -4 * x.abs().double() + 2.0 ** -10 * scale
    assert bool(((k - x).abs() <= step * (1 + 1e-6)).all()) and torch.equal(k, v)
    assert bool(torch.isnan(values(c.pool, HD, fmt)[0][c.bt[0, -1].long(), :, 2:]).all())      # 50 = 3 * 16 + 2: what lies behind is NaN
    assert fields(c.pool, HD)[0].shape == (7, 2, 16, HD)


def test_the_budget_counts_8_bit_pages():
    import dataclasses
    from agens_engine_b200.models import config as Cf
    from agens_engine_b200.serve import budget as B
    cfg = Cf.dense_32b(seed=0)
    k8 = dataclasses.replace(cfg, kv_cache="int8")
    assert cfg.kv_bytes_per_token() == 64 * 2 * 8 * 128 * 2 and k8.kv_bytes_per_token() == 64 * 8 * (2 * 128 + 8) and k8.kv_bytes_per_token(4) == 64 * 2 * 264
    a, b = (B.plan_deployment(c, 24, 262144, 1, 1, 2048, gpu_free_gib=170, host_avail_gib=64) for c in (cfg, k8))
    assert a.host_tier and not b.host_tier and b.fits            # 8-bit pages are not tiered: the context is what the pool holds
    assert b.max_ctx == b.n_pages * 16 > 1.9 * a.n_pages * 16
    kv = B.kv_cache_plan(k8, 262144, 1)
    assert kv == {"extra_bytes": 262144 * 1024 * 4, "split_keys": 1024, "host_tier": False}
    assert B.kv_cache_plan(cfg, 262144, 1, split_keys=64) == {"extra_bytes": 0, "split_keys": 64, "host_tier": True}


def test_the_command_line_takes_a_cache_format(monkeypatch, capsys):
    from agens_engine_b200 import cli
    out = {}
    for fmt in ("bf16", "fp8"):
        assert cli.main(["plan", "--random", "dense-32b", "--budget-gib", "64", "--wctx", "65536", "--kv-cache", fmt, "--host-avail-gib", "8"]) == 0
        out[fmt] = [line for line in capsys.readouterr().out.splitlines() if "KV pool" in line][0]
    pages = {k: int(v.split("KV pool ")[1].split()[0]) for k, v in out.items()}
    assert pages["fp8"] > 1.8 * pages["bf16"]
    monkeypatch.setenv("B200E_KV_CACHE", "int4")
    with pytest.raises(SystemExit, match="kv-cache"):
        cli.main(["plan", "--random", "dense-32b", "--budget-gib", "64"])


def test_a_model_refuses_a_format_that_is_not_there():
    import dataclasses
    from agens_engine_b200.models import config as Cf
    from agens_engine_b200.models.dense import DenseModel
    cfg = Cf.oracle_tiny()
    with pytest.raises(ValueError, match="kv_cache"):
        DenseModel(cfg, "cpu", kv_cache="q8")
    with pytest.raises(ValueError, match="16 tokens"):
        DenseModel(dataclasses.replace(cfg, page_size=32), "cpu", kv_cache="int8")
    with pytest.raises(ValueError, match="heads of 64 or 128"):
        DenseModel(dataclasses.replace(cfg, head_dim=32), "cpu", kv_cache="fp8")
