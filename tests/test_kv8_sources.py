"""Rules of the 8-bit KV kernels that are checked on their sources: what breaks them is a race that no run shows surely."""
import re
from pathlib import Path

import pytest

from tests.test_kernel_sources import _close, _code

SM100 = Path(__file__).resolve().parent.parent / "csrc" / "kernels" / "sm100"


def _body(path, name):
    s = _code(path)
    m = re.search(rf"__global__[^;{{]*\b{name}\s*\(", s)
    i = s.index("{", _close(s, m.end() - 1, "()"))
    return s[i:_close(s, i, "{}")]


@pytest.mark.parametrize("file,kernel", [("kv8_attn.cu", "kv8_attn_kernel"), ("kv8_store.cu", "kv8_store_kernel"), ("kv8_store.cu", "kv8_read_kernel")])
def test_every_block_waits_before_it_lets_dependents_start(file, kernel):
    """No block leaves, reads or lets dependents start before the kernels in front of it are done.  The join rests on it: it reads groups
    and positions before its own wait, which no kernel in front of the attention may still be writing."""
    body = _body(SM100 / file, kernel)
    assert body.count("pdl_wait()") == 1 and body.count("pdl_launch_dependents()") == 1
    before = body[:body.index("pdl_wait()")]
    assert not re.search(r"\breturn\b|\ba\.\w|\bif\b|\bfor\b|pdl_launch_dependents", before), before
    # at the kernel's own level, not inside a branch
    assert before.count("{") - before.count("}") == 1


def test_the_join_reads_no_more_than_groups_before_its_wait():
    path = SM100 / "kv8_attn.cu"
    body = _body(path, "kv8_join_kernel")
    before = body[:body.index("pdl_wait()")]
    assert set(re.findall(r"\ba\.(\w+)", before)) <= {"hq"} and before.count("group_at(a") == 1 and "return" not in before
    s = _code(path)
    i = s.index("Group group_at(")
    fn = s[s.index("{", i):_close(s, s.index("{", i), "{}")]
    assert set(re.findall(r"\ba\.(\w+)\s*\[", fn)) == {"grp_tok0", "grp_cnt", "tok_seq", "tok_pos"} and "status" not in fn
    # and the join follows the attention directly: nothing is launched between them
    run = s[s.index("int run(const Kv8AttnArgs"):]
    launches = re.findall(r"launch\((\w+)", run[:_close(run, run.index("{"), "{}")])
    assert launches == ["kernel", "kv8_join_kernel"]
