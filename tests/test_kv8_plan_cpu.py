"""What a deployment plans for an 8-bit key-value cache and what its model is built with, without a GPU."""
import dataclasses

import pytest
import torch

from agens_engine_b200 import cli
from agens_engine_b200.models import config as C
from agens_engine_b200.models.dense import DenseModel
from agens_engine_b200.ops import kv8 as K
from agens_engine_b200.serve import budget as B


class Built(Exception):
    pass


def _serve(monkeypatch, argv):
    """Runs `serve` up to the model's construction: its arguments, and the deployment that was planned (None without a budget)."""
    got, plan = {}, []

    def init(mc, dev, seed, **kw):
        got.update(kw)
        raise Built
    real = B.plan_deployment
    monkeypatch.setattr(DenseModel, "random_init", staticmethod(init))
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda d=None: (170 << 30, 180 << 30))
    monkeypatch.setattr(B, "cap_process", lambda *a: None)
    monkeypatch.setattr(B, "plan_deployment", lambda *a, **kw: plan.append(real(*a, **kw)) or plan[-1])
    with pytest.raises(Built):
        cli.main(["serve", "--random", "dense-32b", *argv])
    return got, plan[0] if plan else None


@pytest.mark.parametrize("wctx", [4096, 8192, 40000, 131072])
@pytest.mark.parametrize("mode,batch", [("personal", 1), ("server", 8), ("server", 1)])
def test_the_servers_split_is_the_planned_one(monkeypatch, mode, batch, wctx):
    """Sequences that decode together count, not the slots that hold parked ones."""
    argv = ["--kv-cache", "int8", "--mode", mode, "--wctx", str(wctx), "--max-batch", str(batch)]
    got, _ = _serve(monkeypatch, argv)
    assert got["max_seqs"] > batch and got["kv_split"] == K.split_keys_for(wctx, 8 * batch)
    budgeted, dep = _serve(monkeypatch, argv + ["--budget-gib", "100"])
    assert budgeted["kv_split"] == dep.split_keys == got["kv_split"]


def test_short_contexts_of_one_conversation_get_short_splits(monkeypatch):
    got = [_serve(monkeypatch, ["--kv-cache", "fp8", "--mode", "personal", "--wctx", str(n)])[0]["kv_split"] for n in (4096, 8192, 20000, 65536)]
    assert got == [128, 256, 512, 768]


def test_bf16_models_are_built_as_before(monkeypatch):
    got, _ = _serve(monkeypatch, ["--mode", "personal", "--wctx", "8192"])
    assert got == dict(max_seqs=65, max_ctx=8192, prefill_chunk=256, split_keys=64, kv_cache="bf16")


def test_a_plan_names_its_split():
    k8 = dataclasses.replace(C.dense_32b(seed=0), kv_cache="int8")
    plan = lambda batch, slots, tp=1, **kw: B.plan_deployment(k8, 100, 8192, batch, slots, 2048, tp=tp, gpu_free_gib=170, host_avail_gib=64, **kw).split_keys
    assert plan(1, 65) == plan(1, 1) == plan(8, 72, together=1) == 256 and plan(8, 72) == 768 and plan(8, 72, tp=8) == 256
    assert B.plan_deployment(C.dense_32b(seed=0), 100, 8192, 1, 1, 2048, gpu_free_gib=170, host_avail_gib=64, split_keys=64).split_keys == 64


def test_a_model_takes_its_split_and_refuses_others():
    cfg = C.oracle_tiny()
    for bad in (0, 24, 4096, -16):
        with pytest.raises(ValueError, match="kv_split"):
            DenseModel(cfg, "cpu", kv_cache="int8", kv_split=bad)
    with pytest.raises(ValueError, match="kv_split"):
        DenseModel(cfg, "cpu", kv_split=128)


@pytest.mark.parametrize("wctx", [100, 8192, 131072])
@pytest.mark.parametrize("batch,slots,rows", [(1, 65, 128), (8, 72, 128), (1, 1, 32), (2, 6, 48), (20, 20, 128)])
def test_a_plan_counts_the_workspace_that_the_model_has(wctx, batch, slots, rows):
    """The model's step workspace holds eight rows a slot, parked ones included; the planner counts eight a sequence of the batch."""
    k8 = dataclasses.replace(C.dense_32b(seed=0), kv_cache="int8")
    plan = lambda n, c=k8: B.plan_deployment(c, 100, wctx, batch, n, 2048, gpu_free_gib=170, host_avail_gib=64)
    dep, least = plan(slots), plan(batch)
    beyond = dep.plan["fixed_bytes"] - least.plan["fixed_bytes"]
    floats = K.part_floats(rows, 64, 128, wctx, dep.split_keys)
    assert beyond + dep.plan["scratch"]["attention_partials"] >= 4 * floats
    assert beyond == 4 * K.part_floats(rows - min(128, max(32, 8 * batch)), 64, 128, wctx, dep.split_keys)
    assert plan(slots, C.dense_32b(seed=0)).plan["fixed_bytes"] == plan(batch, C.dense_32b(seed=0)).plan["fixed_bytes"]


def test_the_plan_command_counts_the_servers_slots(capsys):
    def pages(convs):
        assert cli.main(["plan", "--random", "dense-32b", "--budget-gib", "64", "--wctx", "131072", "--max-batch", "1", "--max-convs", str(convs),
                         "--kv-cache", "int8", "--host-avail-gib", "8"]) == 0
        return int([line for line in capsys.readouterr().out.splitlines() if "KV pool" in line][0].split("KV pool ")[1].split()[0])
    page = 64 * 8 * (32 * 128 + 128)
    assert abs((pages(0) - pages(64)) - 4 * K.part_floats(96, 64, 128, 131072, 768) / page) <= 1


def test_split_sizes_of_many_contexts_are_not_kept():
    """A caller whose context grows by one a step looks up another one every step."""
    for n in range(1, 3000):
        K.split_keys_for(n, 3)
    assert K.split_keys_for.cache_info().currsize <= 256


def test_a_parked_sequence_goes_back_to_its_own_format_only():
    """int8 and fp8 pages have the same shape: the format goes with a parked sequence, and nothing is touched before it is looked at."""
    import types
    touched = []
    m = types.SimpleNamespace(cfg=dataclasses.replace(C.oracle_tiny(), kv_cache="int8"), new_seq=touched.append)
    for other in ("fp8", "bf16"):
        with pytest.raises(ValueError, match="parked"):
            DenseModel.unpark(m, 0, {"len": 3, "kv": torch.zeros(2, 1, 2, 2176, dtype=torch.uint8), "rope_delta": 0, "kv_cache": other})
    assert touched == []


@pytest.mark.parametrize("mode,split", [("personal", 256), ("server", 768)])
def test_the_plan_command_takes_the_servers_split(monkeypatch, mode, split):
    """A personal server decodes one conversation at a time, whatever --max-batch says."""
    from agens_engine_b200.serve import host as H
    got = {}
    real = H.plan
    monkeypatch.setattr(H, "plan", lambda **kw: got.update(kw) or real(**kw))
    argv = ["--random", "dense-32b", "--budget-gib", "64", "--wctx", "8192", "--kv-cache", "int8", "--mode", mode]
    assert cli.main(["plan", *argv]) == 0
    assert got["split_keys"] == split
    assert split == _serve(monkeypatch, argv[2:])[0]["kv_split"]
