"""Prefix cache: prompts whose page hashes are equal do not share pages."""

import pytest

from axrl_b200.rollout.kv import PyBlockManager, _mix64, make_block_manager

M = (1 << 64) - 1
P = 4


def _unshift(z, k):
    x = z
    for _ in range(64 // k + 1):
        x = z ^ (x >> k)
    return x


def _last_token(h, goal):
    """v with mix(h, v) == goal: every step of the mix is one to one in v."""
    z = _unshift(goal, 31)
    z = z * pow(0x94D049BB133111EB, -1, 1 << 64) & M
    z = _unshift(z, 27)
    z = z * pow(0xBF58476D1CE4E5B9, -1, 1 << 64) & M
    z = _unshift(z, 30)
    v = ((z ^ h) - 0x9E3779B97F4A7C15 - (h << 6 & M) - (h >> 2)) & M
    return v - (1 << 64) if v >> 63 else v


def _state(tokens):
    h = 0
    for t in tokens:
        h = _mix64(h, t & M)
    return h


A = [11, 12, 13, 14]
B = [21, 22, 23]
B.append(_last_token(_state(B), _state(A)))
CHILD = [31, 32, 33, 34]


@pytest.fixture(params=["native", "python"])
def manager(request):
    def make(pages):
        bm = make_block_manager(pages, P) if request.param == "native" else PyBlockManager(pages, P)
        assert type(bm).__name__ == ("BlockManager" if request.param == "native" else "PyBlockManager")
        return bm

    return make


def _match(bm, tokens):
    pages, n = bm.match_prefix(tokens)
    bm.release(pages)
    assert n == len(pages) * P
    return list(pages)


def test_the_two_prompts_collide():
    assert A != B and _state(A) == _state(B)


def test_equal_hashes_are_not_the_same_prompt(manager):
    bm = manager(8)
    a = bm.allocate(2)
    bm.insert(A + CHILD, a)
    assert _match(bm, A + CHILD + [1]) == a
    assert _match(bm, B + CHILD) == [] and _match(bm, B) == []


def test_what_follows_a_collision_is_not_registered(manager):
    """A's page is cached; the page behind B's must not be found behind it."""
    bm = manager(8)
    a = bm.allocate(1)
    bm.insert(A, a)
    b = bm.allocate(2)
    bm.insert(B + CHILD, b)
    assert _match(bm, A + CHILD) == a and _match(bm, B + CHILD) == []
    assert bm.num_cached() == 1
    bm.release(b)
    assert bm.num_free() == 7


def test_pages_behind_an_evicted_one_stay_with_their_prompt(manager):
    bm = manager(4)
    a = bm.allocate(2)
    bm.insert(A + CHILD, a)
    bm.release(a)
    held = bm.allocate(3)  # the two free pages and A's first
    assert bm.num_cached() == 1 and _match(bm, A + CHILD) == []
    bm.insert(B, held[:1])
    assert _match(bm, B + CHILD) != [a[1]] and _match(bm, A + CHILD) == []
    bm.insert(A, held[1:2])  # A's first page again: what hung on it is found again
    assert _match(bm, A + CHILD) == [held[1], a[1]] and _match(bm, B + CHILD) == []
    bm.release(held)
    bm.clear_cache()
    assert bm.num_cached() == 0 and bm.num_free() == 4 and _match(bm, A + CHILD) == []


def test_everything_evicted_leaves_room_for_the_other_prompt(manager):
    bm = manager(3)
    a = bm.allocate(2)
    bm.insert(A + CHILD, a)
    bm.release(a)
    held = bm.allocate(3)
    assert bm.num_cached() == 0
    bm.insert(B + CHILD, held[:2])
    assert _match(bm, B + CHILD) == held[:2] and _match(bm, A + CHILD) == []
    with pytest.raises((IndexError, RuntimeError)):
        bm.insert(B, [99])
