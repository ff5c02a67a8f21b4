"""Where attention over a shared prefix is taken for tree attention, at sizes whose times were
measured, on both sides."""
import pytest


@pytest.mark.parametrize("tokens,heads,requests,groups,positions,want", [
    # one token a request
    (16, 16, 16, 1, 2048, False), (64, 16, 64, 1, 2048, True), (128, 16, 128, 1, 2048, True),
    (128, 16, 128, 1, 1024, True), (64, 8, 64, 1, 2048, True), (64, 16, 64, 1, 1024, False),
    (64, 64, 64, 1, 2048, False), (128, 64, 128, 1, 2048, True), (128, 64, 128, 1, 1024, False),
    (512, 64, 512, 1, 1024, True),
    # drafted tokens
    (64, 16, 8, 1, 1536, False), (128, 64, 64, 1, 2048, False), (256, 64, 128, 1, 2048, False),
    (320, 64, 160, 1, 256, True), (512, 64, 256, 1, 2048, True), (512, 8, 64, 1, 2048, False),
    # groups of four, of two, of one
    (320, 16, 160, 40, 2048, True), (520, 16, 260, 130, 1024, True), (160, 16, 160, 160, 2048, False),
    (320, 64, 160, 160, 2048, False), (64, 16, 64, 64, 2048, False),
    # no token, no request
    (0, 16, 4, 1, 2048, False), (4, 16, 0, 0, 2048, False)])
def test_pays(pkg, tokens, heads, requests, groups, positions, want):
    assert pkg.mla_prefix.pays(tokens, heads, requests, groups, positions) is want
