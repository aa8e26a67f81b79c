"""The numbers by which the workgroups of a scan know a link as one of their own launch (CPU only)."""
import ctypes as ct
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("launches") / "scan_launches.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-shared", "-fPIC", os.path.join(HERE, "scan_launches.cpp"), "-o", path], check=True)
    lib = ct.CDLL(path)
    lib.tag.restype, lib.tag.argtypes = ct.c_uint, [ct.c_ulonglong]
    lib.next.restype, lib.next.argtypes = ct.c_ulonglong, [ct.c_ulonglong]
    lib.after.restype, lib.after.argtypes = ct.c_ulonglong, [ct.c_ulonglong] * 2
    return lib


def test_no_launch_has_the_number_of_words_that_nobody_has_written(launches):
    """From the first launch on, and around 2^32 launches, where a number of 32 bits is used again."""
    for first in (0, (1 << 32) - 1000):
        tags, launch = [], first
        for _ in range(2000):
            tags.append(launches.tag(launch))
            launch = launches.next(launch)
        assert 0 not in tags
        assert len(set(tags)) == 2000, 'launches that follow each other have numbers of their own'


def test_a_number_comes_back_after_all_the_others(launches):
    before = launches.after(1000, (1 << 32) - 2)
    assert launches.tag(before) != launches.tag(1000) == launches.tag(launches.next(before))


def test_a_launch_and_a_place_fit_a_word(launches):
    """A tile's counter has the launch above 28 bits of places."""
    assert launches.next((1 << 32) - 2) < (1 << 32) - 1 < 1 << 36
