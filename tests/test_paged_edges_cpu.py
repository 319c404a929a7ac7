"""CPU tests of the paged cache's boundary: calls that are almost empty (the checks run on the host, before anything is enqueued)."""
import pytest

from tests.test_paged_cpu import append, attend, read, ragged, refused


@pytest.mark.parametrize("call", [append, attend])
@pytest.mark.parametrize("batch,tokens", [(0, 3), (3, 0)])
def test_without_offsets_rows_and_sequences_are_the_same_number_also_when_one_is_none(call, batch, tokens):
    assert refused(call(batch=batch, tokens=tokens), "one row per sequence")
    assert call(batch=batch, tokens=tokens, cu=1 << 20) == 0


def test_calls_without_sequences_or_rows_do_nothing():
    assert append(batch=0, tokens=0) == 0 and attend(batch=0, tokens=0) == 0
    assert read(batch=0) == 0 and read(rows=0) == 0 and ragged(batch=0) == 0 and ragged(tokens=0) == 0
