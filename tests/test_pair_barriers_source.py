"""Barriers that one block of a pair arrives at and the other waits for order memory only in the scope of their
cluster. No run on one GPU shows a scope that is too small, so the source is held against it."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "arcqml_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def test_barrier_instructions_name_their_scope():
    text = source("tensor_core.cuh")
    waits = re.findall(r"mbarrier\.(?:try_wait|test_wait)[.\w:]*", text)
    arrivals = re.findall(r"mbarrier\.arrive\.(?!expect_tx)[.\w:]*", text)
    assert waits and arrivals
    for found in waits + arrivals:
        assert re.search(r"\.(?:acquire|release|relaxed)\.(?:cta|cluster)\.", found), found
    # one form of each for a block, one for a pair
    for found in (waits, arrivals):
        assert {".cluster." in re.sub(r"shared::\w+", "", f) for f in found} == {True, False}
    # a relaxed arrival releases by the fence before it
    for i in (m.start() for m in re.finditer(r"mbarrier\.arrive\.relaxed", text)):
        assert "fence.release.sync_restrict::shared::cta.cluster" in text[i - 120:i]


def test_barriers_of_a_pair_are_waited_for_in_its_scope():
    text = source("muon.cu")
    kernel = text[text.index("    k_product(const __grid_constant__ Group g"):text.index("// A wait that ran out left")]
    waits = re.findall(r"wait_for(<\w+>)?\(&st\.(\w+)", kernel)
    assert {b for _, b in waits} == {"empty", "full", "taken", "peer", "done"}
    for scope, barrier in waits:
        # only a block's own copies arrive at `full`
        assert scope == ("<1>" if barrier == "full" else "<CG>"), (scope, barrier)
    arrivals = re.findall(r"barrier_arrive_at(<\w+>)?\(", kernel)
    assert arrivals and set(arrivals) == {"<CG>"}


def test_a_block_stays_until_its_last_stages_are_read():
    """The tensor cores arrive at `empty` of both blocks some time after the products were issued: the thread that
    copies in waits for that behind its last stage, since a block that has ended has no shared memory to arrive in."""
    text = source("muon.cu")
    copies = text[text.index("if (warp == 0 && lane == 0) { // copies operands in"):text.index("// issues the products")]
    loop = copies.index("for (; on && more; more = walk.next(part))")
    behind = copies[copies.index("if (++at == S)", loop):]
    assert re.search(r"if \(on\) wait_for<CG>\(&st\.empty\[s\], s < at \? phase : phase \^ 1", behind)


def test_parities_behind_the_last_stage():
    """`empty` of stage s has gone through as many phases as the stage was filled when what the test above looks for
    passes: a barrier of n phases passes parity (n - 1) & 1, and a fresh one parity 1."""
    for stages in (3, 6):
        at, phase, filled = 0, 0, [0] * stages
        for _ in range(40):
            for s in range(stages):
                parity = phase if s < at else phase ^ 1
                assert parity == (filled[s] - 1) & 1
            filled[at] += 1
            at += 1
            if at == stages:
                at, phase = 0, phase ^ 1
