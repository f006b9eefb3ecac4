"""Where the copies of forks live."""


def test_row_copies_are_in_the_library_that_every_engine_loads():
    from gibbs_b200.csrc.build import LIBRARIES
    from gibbs_b200.ops import row_copies
    from gibbs_b200.ops.library import library
    assert row_copies.LIBRARY == "core" and "row_copies.cu" in LIBRARIES["core"]
    assert library("core").gb_row_copies_piece_bytes() == 4096
