"""Losses on the CPU: refusals and host-side settings beyond those of test_losses.py."""


def test_tries_of_the_waits_are_bounded_and_put_back(pkg):
    before = pkg.losses_selftest_tries(5)
    assert before > 5
    assert pkg.losses_selftest_tries(0xFFFFFFFF) == 5
    assert pkg.losses_selftest_tries(before) == before          # no more than the number they start with
