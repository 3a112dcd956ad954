"""The gated delta rule's forward keeps within the workspace whose size the library names: for every
type, with and without a state that is handed on, the bytes that the call lays its parts out in,
counted here from the layout itself.

A chunk of 64 steps of a value head keeps three rows of 64 float32 and two triangles of six operands
of 64 x 8 values, the first one once for each of the operands' parts; where the scan has few blocks a
chunk of a key head keeps 12 operands for every 32 keys beside them.  The chunks are prepared in the
fewest equal parts within 192 MiB, and several parts hand each other the state."""

import random

import pytest

import oxide_hip as ox

SIZES = {ox.F32: 4, ox.BF16: 2}


def up(v, to):
    return (v + to - 1) // to * to


def used(batch, time, key_heads, heads, keys, values, element, parts):
    """(bytes, parts of the sequence)."""
    operand, slabs = 64 * 8 * element, (values + 15) // 16
    head = batch * heads * (3 * 64 * 4 + 6 * parts * operand + 6 * operand)
    many = batch * heads * ((slabs + 1) // 2) >= 256
    key = 0 if many else batch * key_heads * (up(keys, 32) // 32) * 12 * operand
    chunks = (time + 63) // 64
    most = max(1, (192 << 20) // (head + key))
    count = (chunks + most - 1) // most
    each = (chunks + count - 1) // count
    state = up(batch * heads * keys * values * 4, 256) if each < chunks else 0
    return up(each * head, 256) + up(each * key, 256) + state, count


def reported(code, dims):
    _, alone, saves, _, _ = ox._delta_plan(code, *dims)
    return alone, saves


def check(dims):
    for code, element in SIZES.items():
        # bfloat16: one part without a final state, two with one; float32 has one
        forms = (1,) if code == ox.F32 else (1, 2)
        needs = max(used(*dims, element, parts)[0] for parts in forms)
        alone, saves = reported(code, dims)
        assert saves >= needs, (dims, code, saves, needs)
        assert alone == 0 or alone >= needs, (dims, code, alone, needs)


@pytest.mark.parametrize("batch,time,heads", [
    (8, 6144, 16), (8, 4096, 24), (4, 8192, 24), (1, 24576, 16), (16, 2688, 16), (1, 12160, 16)])
def test_training_and_prompts_in_parts(batch, time, heads):
    check((batch, time, heads, heads, 128, 128))


@pytest.mark.parametrize("batch,key_heads,heads,keys,values", [
    (1, 16, 16, 128, 128), (8, 16, 16, 128, 128), (3, 1, 4, 17, 40), (64, 8, 16, 32, 8),
    (1, 1, 1, 64, 16), (2, 4, 12, 96, 200)])
def test_around_every_change_of_the_parts(batch, key_heads, heads, keys, values):
    """The lengths at which one form or the other begins to take another part, and their neighbours."""
    ends = {64}
    for element in (2, 4):
        for parts in (1, 2):
            def count_of(chunks):
                return used(batch, 64 * chunks, key_heads, heads, keys, values, element, parts)[1]

            last = 1
            for count in (1, 2, 3, 4):  # the last length of so many parts
                low, high = last, 2 * last
                while count_of(high) <= count:
                    high *= 2
                while high - low > 1:
                    at = (low + high) // 2
                    low, high = (low, at) if count_of(at) > count else (at, high)
                ends.update(64 * c + d for c in (low, high) for d in (-63, -1, 0, 1))
                last = high
    for time in sorted(ends):
        if batch * heads * ((time + 63) // 64) <= 1 << 23:
            check((batch, time, key_heads, heads, keys, values))


def test_shapes_at_random():
    r = random.Random(5)
    for _ in range(3000):
        key_heads, group = r.choice([1, 2, 3, 8, 16, 32]), r.choice([1, 1, 2, 3, 4])
        batch = int(2 ** r.uniform(0, 8))
        time = int(2 ** r.uniform(0, 17))
        if batch * key_heads * group * ((time + 63) // 64) > 1 << 23:
            continue  # more than one call takes
        check((batch, time, key_heads, key_heads * group, r.randint(1, 128),
               r.choice([8, 16, 64, 128, 256, r.randint(1, 512)])))
