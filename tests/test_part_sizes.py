"""Workspaces of the calls on caller-owned memory that verify drafted tokens or attend with sinks and prefixes: one that serves a
loop's largest call serves its smaller ones. (No device is touched.)"""
import itertools


def growing(sizes):
    """Neighbours of a grid of sizes, the second no smaller anywhere."""
    for at in itertools.product(*(range(len(s)) for s in sizes)):
        for i, s in enumerate(sizes):
            if at[i] + 1 < len(s):
                more = at[:i] + (at[i] + 1,) + at[i + 1:]
                yield tuple(s[k] for s, k in zip(sizes, at)), tuple(s[k] for s, k in zip(sizes, more))


def test_verification_of_fewer_tokens_needs_no_more(gq):
    for small, large in growing(([1, 2, 3, 7, 8, 12, 13, 16, 31, 32, 33, 64, 500, 1000], [0, 1, 3, 4, 5, 31, 32], [1, 7, 2048, 2049, 4096, 4097, 32003, 151936, 1 << 20])):
        assert 0 < gq.draft_work(*small) <= gq.draft_work(*large), (small, large)
