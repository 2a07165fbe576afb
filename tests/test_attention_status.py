"""Status codes and the count of tries of a wait: what needs no GPU."""
from so3lr_b200._lib import STATUS, So3lrB200Error, lib


def test_codes_have_their_words():
    for code, words in STATUS.items():
        assert lib.so3lr_b200_status_string(code).decode() == words
    assert sorted(STATUS) == list(range(7)) and "wait" in str(So3lrB200Error(6, "structure_attention"))


def test_tries_of_a_wait():
    before = lib.so3lr_b200_host_wait_tries(-1)
    try:
        assert before == 500000 and lib.so3lr_b200_host_wait_tries(7) == -1
    finally:
        assert lib.so3lr_b200_host_wait_tries(before) == 7
    assert lib.so3lr_b200_host_wait_tries(before) == before
