"""The workspace of a decode over spans holds the states of parts that can be, not of every part
of every row of the tables: these queries need no GPU."""

from __future__ import annotations

import pytest

pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from heteroserve import _hip

    if not _hip.lib_path().exists():
        pytest.fail(f"{_hip.lib_path()} missing: run python hetero-serve_amd/build.py")
    return _hip.open_library()


def _bytes(lib, kv, B, H, Hkv, D, tokens):
    if kv == "q4":
        return lib.hs_q4_decode_workspace_bytes(B, H, Hkv, D, 16, tokens // 16, 0, 0)
    return lib.hs_window_decode_workspace_bytes(kv, B, H, Hkv, D, 16, tokens // 16, 0, 0)


@pytest.mark.parametrize("kv,keys", [("q4", 2048), (1, 1024), (2, 1024)])
@pytest.mark.parametrize("H,Hkv,D", [(32, 8, 128), (16, 16, 64), (8, 8, 32)])
@pytest.mark.parametrize("B", [3, 64, 256])
@pytest.mark.parametrize("tokens", [2 ** 17, 2 ** 20])
def test_wide_tables(lib, kv, keys, H, Hkv, D, B, tokens):
    """Parts are fitted: fewer than `keys` keys each, the longest that they become, only while few
    enough to be on the chip together."""
    state = H * (4 * D + 8)
    most = B * (tokens // keys) * state + 8 * B + 16
    assert 0 < _bytes(lib, kv, B, H, Hkv, D, tokens) <= most
    assert most < 0.6 * B * (tokens // (keys // 4)) * state


@pytest.mark.parametrize("kv", ["q4", 1, 2])
def test_more_rows_than_are_fitted(lib, kv):
    """Parts grow with the table rather than the workspace past 256 MiB, up to the longest."""
    for tokens in (2 ** 13, 2 ** 15, 2 ** 17):
        longest = 2048 if kv == "q4" else 1024
        need = _bytes(lib, kv, 512, 32, 8, 128, tokens)
        assert 0 < need <= max(2 ** 28, 512 * (tokens // longest) * 32 * 520)
