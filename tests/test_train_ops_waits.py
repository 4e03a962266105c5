"""What the kernels of the training operators leave after a wait that ran out, read from their sources: no test makes one run out in
a kernel, and a kernel that gave up must not look like one that has finished."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "litnicelm_b200", "csrc")
WAIT = r"(?:mbar_wait\w*|TF_WAIT)\("
AGREED = "ok = __all_sync(0xffffffffu, ok && !*abort_flag);"


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    return re.sub(r"//[^\n]*", "", text)


def body_of(text, name):
    """What stands between the braces of a function."""
    m = re.search(r"\b" + name + r"\([^{};]*\)\s*\{", text)
    assert m, name
    depth, at = 1, m.end()
    while depth:
        depth += {"{": 1, "}": -1}.get(text[at], 0)
        at += 1
    return text[m.end():at]


@pytest.mark.parametrize("file,store,names", [
    ("train_attention_tc.cu", "tt_store_row(",
     ("train_forward_tc_kernel", "train_forward_pair_kernel", "train_dkv_tc_kernel", "train_dq_tc_kernel")),
    ("train_attention_f32.cu", "tf_store_sums(", ("train_forward_f32_kernel", "tf_dkv", "tf_dq"))],
    ids=lambda x: x if isinstance(x, str) and x.endswith(".cu") else "")
def test_attention_stores_behind_the_flag(file, store, names):
    """Between the last wait and the results every warp asks whether any has given up: a barrier that another role completes while
    it gives up (the tensor pipe's last) says nothing about the sums."""
    for name in names:
        body = body_of(source(file), name)
        at = body.index(store)
        waits = [m.start() for m in re.finditer(WAIT, body[:at])]
        assert waits and AGREED in body[waits[-1]:at], name


def test_attention_forward_drains_on_its_own_barrier():
    body = body_of(source("train_attention_tc.cu"), "train_forward_tc_kernel")
    drain = body[body.index("if (!ok) {"):]
    drain = drain[:drain.index("}\n")]
    (bar,) = re.findall(r"tc_commit\((\w+)\)", drain)
    assert not re.search(WAIT + bar + r"\b", body), bar


def test_policy_rows_behind_a_lost_one():
    """A row whose copy is late leaves the barrier in a phase of its own: the rows after it must not wait there, nor ask for copies,
    and the copy must land before the shared memory goes away."""
    body = body_of(source("policy_loss.cu"), "policy_stream_kernel")
    loop = body[body.index("for (int row = blockIdx.x"):]
    wait = re.search(WAIT, loop).start()
    assert re.search(r"if \(lost\) \{\s*fill_row<T>\(a, w, f, row, NAN, tid, THREADS\);\s*continue;", loop[:wait])
    assert re.search(r"lost = !__syncthreads_and\(there\);\s*if \(lost\) \{\s*fill_row<T>\(a, w, f, row, NAN, tid, THREADS\);\s*continue;", loop[wait:])
    assert all("!lost" in loop[loop.rindex("if", 0, m.start()):m.start()] for m in re.finditer(r"fetch\(after", loop[:wait]))
    assert re.search(r"if \(lost && tid == 0\) \{[^}]*mbar_try_wait\(bar, \(phase - 1u\) & 1u\) && global_timer\(\) < limit", loop[wait:])
