"""Expired waits in the pointwise convolutions' kernels, read from their sources: a thread learns of a loss by itself, so
its partners at a barrier need not know.  A loop is left on a loss only by a thread that works alone (`lane == 0`), or by a
whole warp (`__any_sync`) whose loop has no other warps' barriers; elsewhere one thread would go on to the kernel's last
barrier while its partners waited at the loop's."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "box-convolutions_b200", "csrc")
# a jump or a wait that depends on a loss
ON_LOSS = re.compile(r"if \([^;\n]*(?:!wait\(|wait\.lost)[^;\n]*\) (?:break|return|continue|wait\()")
OTHER_WARPS = re.compile(r"bar\.sync|__syncthreads|together\(")


def without_comments(text):
    return re.sub(r"//[^\n]*", "", text)


def scopes(text):
    """(start, end, what stands in front of it) of every pair of braces."""
    text = re.sub(r"\w\{[^{};]*\}", lambda m: " " * len(m.group()), text)      # (initial values)
    open_at, out, start, depth = [], [], 0, 0
    for m in re.finditer(r"[(){};]", text):
        c = m.group()
        depth += (c == "(") - (c == ")")
        if c in "()" or c == ";" and depth:
            continue
        if c == "{":
            open_at.append((m.start(), text[start:m.start()], depth))
            depth = 0
        elif c == "}" and open_at:
            begin, head, depth = open_at.pop()
            out.append((begin, m.end(), head))
        start = m.end()
    return out


def shared_exits(text):
    text = without_comments(text)
    places = scopes(text)
    found = []
    for m in ON_LOSS.finditer(text):
        around = [p for p in places if p[0] < m.start() < p[1]]
        if any(re.search(r"\blane == 0\b", head) for _, _, head in around):
            continue
        loops = [text[a:b] for a, b, head in around if re.search(r"\b(for|while|do)\b", head)]
        if "__any_sync" in m.group() and loops and not any(OTHER_WARPS.search(t) for t in loops):
            continue
        found.append(text[:m.start()].count("\n") + 1)
    return found


@pytest.mark.parametrize("name", ["pointwise_mma.cu", "pointwise_split.cu"])
def test_only_a_thread_alone_leaves_its_loop_on_a_loss(name):
    text = open(os.path.join(CSRC, name)).read()
    assert len(ON_LOSS.findall(without_comments(text))) >= 4      # (of the threads that issue copies and products)
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
    warp = "void f() { for (;;) { if (__any_sync(all, !wait(full, 0))) break; __syncwarp(); } }"
    pair = "void f() { for (;;) { if (__any_sync(all, wait.lost)) break; together(); } }"
    assert shared_exits(alone) == [] and shared_exits(shared) == [1] and shared_exits(warp) == [] and shared_exits(pair) == [1]
