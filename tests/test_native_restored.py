"""CPU: what one test puts in the place of the native call path does not reach the next."""
from ferret_amd import lib

NATIVE = lib.native


def test_one_replaces_it():
    lib.native = lambda: lib._Absent()


def test_the_next_has_the_librarys():
    assert lib.native is NATIVE
