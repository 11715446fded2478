"""Runs the C++ test of a block's operators (tests/cpp/test_block_operators.cpp) on the GPU, also as a
host-side AddressSanitizer/UBSan build; see tests/test_cpp_dropin.py."""
import pytest

import test_cpp_dropin

pytestmark = pytest.mark.gpu


def test_block_operators_through_the_cpp_store():
    test_cpp_dropin.test_cpp_dropin("test_block_operators")


def test_block_operators_through_the_cpp_store_host_sanitizers():
    test_cpp_dropin.test_cpp_dropin_host_sanitizers("test_block_operators")
