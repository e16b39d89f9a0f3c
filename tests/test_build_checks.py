"""What the build looks for in the listing of the grouped products' tiles (build.check_piece_lines)."""

import importlib.util
import os

import pytest


def _build():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nki-library_amd", "build.py")
    spec = importlib.util.spec_from_file_location("moe_build", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


GOOD = ["v_add3_u32 v2, s79, v229, v228", "ds_write_b128 v2, v[4:7]", "ds_write_b128 v8, v[4:7] offset:4096", "ds_write_b128 v3, v[4:7]"]


@pytest.mark.parametrize("bad", ["ds_write_b128 v2, v[2:5]", "ds_write_b128 v5, v[2:5] offset:4096", "ds_write_b128 v31, v[30:33] offset:24576"])
def test_a_piece_that_holds_its_address_is_found(bad):
    build = _build()
    build.check_piece_lines(GOOD, "listing")
    with pytest.raises(RuntimeError, match="writes its own address"):
        build.check_piece_lines([*GOOD, bad], "listing")


def test_a_listing_without_pieces_is_not_taken_for_a_good_one():
    with pytest.raises(RuntimeError, match="no piece"):
        _build().check_piece_lines(["s_nop 0", "ds_write_b64 v2, v[2:3]"], "listing")


def test_without_the_listing_tools(tmp_path, monkeypatch):
    monkeypatch.setenv("ROCM_PATH", str(tmp_path))
    build = _build()
    assert "not checked" in build.check_tile_code("x.o", build.check_piece_lines)
