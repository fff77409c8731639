"""CPU: lengths that a call reads and writes must not share memory in part, which threads would race for."""
import pytest

from test_q8_refusals_cpu import P, _append_args, _fill_args


@pytest.mark.parametrize("change", [
    dict(start=P + 64, out=P + 64), dict(start=P + 64, out=P + 68), dict(start=P + 68, out=P + 64), dict(out=P), dict(out=P + 8), dict(out=P - 4)])
def test_fill(lib, change):
    assert lib.ifv2_q8_fill(*_fill_args(**change)) == -1 and b"overlap" in lib.ifv2_last_error()


@pytest.mark.parametrize("change", [
    dict(pos=P + 4), dict(pos=P - 4), dict(pos=P + 8, n1=P + 12), dict(n1=P), dict(n1=P + 8, n2=P + 8, c2=P, cc2=1, k2=1, s2=1)])
def test_append(lib, change):
    assert lib.ifv2_q8_append(*_append_args(**change)) == -1 and b"overlap" in lib.ifv2_last_error()
