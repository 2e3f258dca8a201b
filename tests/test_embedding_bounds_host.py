"""What the lookup entry points refuse at the edges of their arguments, before any CUDA call: see
test_embedding_muon_host.py."""
import pytest

from test_embedding_muon_host import Call


@pytest.fixture
def call(runtime):
    return Call(runtime)


@pytest.mark.parametrize("dtype, data", [(0, 68), (0, 66), (1, 66), (2, 65), (3, 65)])
def test_rows_that_are_none_start_on_an_element_too(call, dtype, data):
    """The width of accesses follows from the addresses, also from that of a table or gradient without rows: off an
    element's boundary it would be less than an element, and the output's end would be passed."""
    none = call.rows(data=data, rows=0, dtype=dtype)
    call.message(call.lookup(table=none, output=call.rows(rows=3, dtype=dtype)), "table is not aligned")
    call.message(call.gradient(gradient=none, output=call.rows(dtype=dtype)), "gradient is not aligned")
    wide = dict(width=40_000, dtype=dtype)
    call.message(call.gradient(gradient=call.rows(data=data, rows=0, **wide), options=call.options(normalize=1),
                               table=call.rows(**wide), output=call.rows(**wide)), "gradient is not aligned")
