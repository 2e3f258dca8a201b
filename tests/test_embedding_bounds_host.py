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


def test_padding_that_is_no_index(runtime):
    """The binding refuses what 8 bytes cannot hold as it refuses a negative one."""
    from types import SimpleNamespace

    class Indices:
        is_cuda, dtype = True, "int64"

        def get_device(self):
            return 0

    fake = SimpleNamespace(Tensor=Indices, int64="int64", int32="int32")
    for padding in (-1, 2 ** 63, 2 ** 70):
        with pytest.raises(ValueError, match="padding index"):
            runtime._embedding_call(fake, Indices(), 1.0, False, padding, 0)
    for padding in (None, 0, 2 ** 63 - 1):
        assert len(runtime._embedding_call(fake, Indices(), 1.0, False, padding, 0)) == 24


def test_messages_name_the_limits(call):
    """2^31 rows are refused, one less is not."""
    call.message(call.lookup(table=call.rows(rows=1 << 31)), "below 2^31")
    # (the next check is reached)
    call.message(call.lookup(table=call.rows(rows=(1 << 31) - 1), output=call.rows(rows=4)), "output")
