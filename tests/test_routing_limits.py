"""Routing of more tokens than a launch has workgroups for is refused before anything touches a GPU."""
from cubek_amd import _ffi, routing
from test_matmul_refusals import CLIENT, ROUTE, status, t


def test_too_many_tokens():
    for tokens, refused in (((1 << 28) - 64, "WORKSPACE_TOO_SMALL"), ((1 << 28) - 63, "TOO_LARGE"), (1 << 31, "TOO_LARGE")):
        a = {**ROUTE, "logits": t(tokens, 8, size=4), "rows": t(2 * tokens, size=4), **{k: t(tokens, 2, size=4) for k in ("weights", "experts", "slots")}}
        assert status(routing.launch_ref, CLIENT, a["logits"], a["weights"], a["experts"], a["offsets"], a["rows"], a["slots"], a["elem"]) == getattr(_ffi, "ERR_" + refused)
    assert routing.workspace_bytes((1 << 28) - 64, 8, 2) > 0 and routing.workspace_bytes((1 << 28) - 63, 8, 2) == 0
