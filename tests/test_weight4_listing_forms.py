"""The listings of the products with weights in 4 bits: the forms that the other checks of them leave out."""

import re

import test_weight4_listing as base
from test_weight4_listing import listing  # noqa: F401


def test_the_large_tiles_of_groups_of_64(tmp_path):
    """A build of its own, with a schedule of its own around the same assembly."""
    base.test_matrix_instructions_do_not_read_what_was_just_written(64, tmp_path)


def test_every_kernel_states_its_memory(listing):  # noqa: F811
    """One line a kernel, so that a check of these lines sees all of them."""
    kernels = re.findall(r"^\s*\.amdhsa_kernel (_Z\d+w4_\w+)", listing, re.M)
    stated = dict(re.findall(r"^(_Z\d+w4_\w+):.*?^; ScratchSize: (\d+)", listing, re.S | re.M))
    assert len(kernels) == 100 and sorted(kernels) == sorted(stated) and set(stated.values()) == {"0"}
