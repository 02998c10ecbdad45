"""Which KV format the multi-token-prediction head of a model with 8-bit pages has, without a GPU."""
import dataclasses
import types

import pytest

from agens_engine_b200.models import config as C
from agens_engine_b200.models import mtp
from agens_engine_b200.parallel import tp_model as T


class Built(Exception):
    pass


def _head(monkeypatch, target, **kw):
    got = {}

    def init(self, cfg, device, **k):
        got.update(k, cfg=cfg)
        raise Built
    monkeypatch.setattr(mtp.DenseModel, "__init__", init)
    with pytest.raises(Built):
        mtp.MtpHead(target, **kw)
    return got


def _target(cfg, kv_cache, split8, **kw):
    return types.SimpleNamespace(cfg=dataclasses.replace(cfg, kv_cache=kv_cache), dev="cpu", max_seqs=5, max_ctx=4096, split_keys=64, split8=split8,
                                 lm_rows=cfg.vocab, **kw)


@pytest.mark.parametrize("kv_cache,split8", [("bf16", None), ("int8", 128), ("fp8", 768)])
@pytest.mark.parametrize("tp", [1, 2])
def test_the_heads_pages_are_the_targets(monkeypatch, kv_cache, split8, tp):
    """On one GPU and beside a shard, whose whole config does not name the format that the shard was built with."""
    cfg = C.dense_32b(seed=0)
    target = _target(cfg, kv_cache, split8) if tp == 1 else _target(T.local_config(cfg, tp), kv_cache, split8, full_cfg=cfg)
    got = _head(monkeypatch, target)
    assert got["kv_cache"] == kv_cache and got.get("kv_split") == split8
    assert got["cfg"].n_kv_heads == 8 and got["cfg"].n_layers == 1 and got["max_seqs"] == 5


def test_a_head_of_another_format(monkeypatch):
    cfg = C.dense_32b(seed=0)
    got = _head(monkeypatch, _target(cfg, "int8", 128), kv_cache="bf16")
    assert got["kv_cache"] == "bf16" and "kv_split" not in got
    got = _head(monkeypatch, _target(cfg, "bf16", None), kv_cache="fp8")
    assert got["kv_cache"] == "fp8" and "kv_split" not in got
