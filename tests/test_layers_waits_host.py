"""Expired waits in the pointwise convolutions' kernels, read from their sources: a thread learns of a loss by itself, so
its partners at a barrier need not know.  A loop is left on a loss only by a thread that works alone (`lane == 0`);
elsewhere one thread would go on to the kernel's last barrier while its partners waited at the loop's."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "box-convolutions_b200", "csrc")
# a jump or a wait that depends on a loss
ON_LOSS = re.compile(r"if \((?:!wait\(.*\)|!?wait\.lost|.*wait\.lost.*)\) (break|return|continue|wait\()")


def scopes(text):
    """(position, headers of the braces that are open there) of every character that opens or closes one."""
    open_at, out, start = [], [], 0
    for m in re.finditer(r"[{};]", text):
        if m.group() == "{":
            open_at.append(text[start:m.start()])
        elif m.group() == "}" and open_at:
            open_at.pop()
        start = m.end()
        out.append((m.end(), list(open_at)))
    return out


def shared_exits(text):
    text = re.sub(r"//[^\n]*", "", text)
    places = scopes(text)
    found = []
    for m in ON_LOSS.finditer(text):
        at = max((p for p in places if p[0] <= m.start()), default=(0, []), key=lambda p: p[0])[1]
        if not any(re.search(r"\blane == 0\b", h) for h in at):
            found.append(text[:m.start()].count("\n") + 1)
    return found


@pytest.mark.parametrize("name", ["pointwise_mma.cu", "pointwise_split.cu"])
def test_only_a_thread_alone_leaves_its_loop_on_a_loss(name):
    text = open(os.path.join(CSRC, name)).read()
    assert len(ON_LOSS.findall(re.sub(r"//[^\n]*", "", text))) >= 4      # (of the threads that issue copies and products)
    assert shared_exits(text) == []


@pytest.mark.parametrize("name", ["pointwise_mma.cu", "pointwise_split.cu"])
def test_a_block_that_lost_an_arrival_waits_before_it_frees_what_products_write(name):
    text = open(os.path.join(CSRC, name)).read()
    ends = [m.start() for m in re.finditer(r"\btmem_free\(", text)]
    assert len(ends) == 2
    for end in ends:
        assert re.search(r"if \(wait\.lost\) let_copies_land\(\);\s+__syncwarp\(\);\s+tmem_release\(\);\s+__syncthreads\(\);[^;]*$", text[:end])


def test_the_reader_finds_a_shared_exit():
    alone = "void f() { if (lane == 0) { for (;;) { if (!wait(full, 0)) break; } } }"
    shared = "void f() { for (;;) { if (!wait(full, 0)) break; __syncwarp(); } }"
    assert shared_exits(alone) == [] and shared_exits(shared) == [1]
