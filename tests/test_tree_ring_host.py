"""The ring of key and value blocks of the tensor-core kernels for drafted tokens, walked through on the host: whatever the order in
which the TMA warp, the warps that issue products, the warp that mends values and the loads themselves get on, nobody waits for good.

A barrier is asked by the parity of a phase, so whoever asks must not be two phases late: a slot may be filled again only once
everyone who asks about it has seen that it was full.  Softmax is left out (P follows S at once): it only delays the products."""
import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(__file__), '..', 'native_sparse_attention_pytorch_b200', 'csrc', 'nsa_tree.cu')


def stuck_states(slots, blocks, streams, mender_frees):
    """-> states without a next step in which someone is not through.  Block 2u is K of block u, 2u + 1 its V; S is two blocks ahead.
    A state: blocks requested, their landing, steps of each product warp, steps of the mending warp."""
    order = []                                       # a product warp's steps: ('s', u) and ('pv', u)
    for u in range(min(2, blocks)):
        order.append(('s', u))
    for u in range(blocks):
        order.append(('pv', u))
        if u + 2 < blocks:
            order.append(('s', u + 2))
    mending = [(kind, u) for u in range(blocks) for kind in ('k', 'v')]
    arrivals = streams + (1 if mender_frees else 0)

    def full(state, i):
        """The phase of block i's slot in which it lands, asked by parity"""
        slot, round_ = i % slots, i // slots
        done = sum(1 for x in range(slot, state[0], slots) if state[1] >> x & 1)
        return done % 2 != round_ % 2

    def released(state, i):
        """Has block i been given back by everyone who counts?"""
        step = order.index(('s', i // 2) if i % 2 == 0 else ('pv', i // 2))
        n = sum(1 for pc in state[2] if pc > step)
        if mender_frees:
            n += 1 if state[3] > mending.index(('k' if i % 2 == 0 else 'v', i // 2)) else 0
        return n == arrivals

    def next_states(state):
        requested, landed, products, mended = state
        i = requested
        if i < 2 * blocks and (i < slots or released(state, i - slots)):
            yield (i + 1, landed, products, mended)
        for x in range(requested):
            if not landed >> x & 1:
                yield (requested, landed | 1 << x, products, mended)
        for s, pc in enumerate(products):
            if pc == len(order):
                continue
            kind, u = order[pc]
            # values are waited for through the mending warp
            ready = full(state, 2 * u) if kind == 's' else mended > mending.index(('v', u))
            if ready:
                yield (requested, landed, products[:s] + (pc + 1,) + products[s + 1:], mended)
        if mended < len(mending):
            kind, u = mending[mended]
            if full(state, 2 * u + (kind == 'v')):
                yield (requested, landed, products, mended + 1)

    start = (0, 0, (0,) * streams, 0)
    seen, todo, stuck = {start}, [start], []
    while todo:
        state = todo.pop()
        after = list(next_states(state))
        if not after and (state[0] < 2 * blocks or state[3] < len(mending) or min(state[2]) < len(order)):
            stuck.append(state)
        for s in after:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return stuck


def mender_frees():
    """Does the mending warp give blocks back, and is it counted, in both kernels?"""
    with open(SOURCE) as f:
        text = f.read()
    counts = re.findall(r'mbar_init\(smem_u32\(&bars\.free\[i\]\), ([^)]*)\)', text)
    assert len(counts) == 2
    role = text[text.index('void mend_blocks('):text.index('tree_tc_kernel(')]
    gives = len(re.findall(r'mbar_arrive\(smem_u32\(&bars\.free\[', role))
    assert (gives, counts) in ((0, ['streams', '1']), (2, ['streams + 1', '2'])), (gives, counts)
    return gives == 2


SHAPES = [(4, 5, 1), (5, 6, 1), (6, 6, 1), (4, 4, 2), (5, 4, 2)]


@pytest.mark.parametrize('slots, blocks, streams', SHAPES)
def test_nobody_waits_for_good(slots, blocks, streams):
    assert not stuck_states(slots, blocks, streams, mender_frees())


@pytest.mark.parametrize('slots, blocks, streams', SHAPES[:3])
def test_the_walk_finds_a_ring_that_the_mending_warp_has_no_part_in(slots, blocks, streams):
    """Keys given back by the products alone: their slot may be full again before the mending warp has asked about it."""
    assert stuck_states(slots, blocks, streams, False)
