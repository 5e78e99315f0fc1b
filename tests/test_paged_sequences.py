"""What the Python calls on sequences of different lengths take for `Sequences`: tables as they lie in memory."""
import numpy as np
import pytest
import torch

from ratchet_amd import Device, OperationError, Sequences, Tensor

CPU = Device.CPU


def zeros(*shape, dt=np.float16):
    return Tensor.from_data(np.zeros(shape, dt))


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


# ---- tables: a row lies table_stride entries behind the one before, and each has its width, in its own memory


def overlapping():
    line = torch.arange(8, dtype=torch.int32)
    return {
        "one row for all": line[None, :4].expand(2, 4), "rows one apart": line.unfold(0, 4, 1)[:2], "rows three apart": line.as_strided((2, 4), (3, 1)),
        "the last row at the storage's end": line[:5].unfold(0, 4, 1), "one entry for all": line[:1, None].expand(2, 1).as_strided((2, 1), (0, 1)),
    }


@pytest.mark.parametrize("name", list(overlapping()))
def test_tables_whose_rows_overlap_are_refused(name):
    """Read with rows their width apart, they would be read past their storage."""
    table = overlapping()[name]
    pool = Tensor.empty_cache((6, 2, 16, 64), CPU)
    seqs = Sequences(2, ints(0, 3, 4), 3, ints(5, 6), table)
    with pytest.raises(OperationError, match="table"):
        pool.cache_write_paged(zeros(4, 128), seqs)
    with pytest.raises(OperationError, match="table"):
        zeros(4, 512).attention_paged(pool, pool, seqs)


@pytest.mark.parametrize("table,stride", [
    (torch.zeros((2, 4), dtype=torch.int32), 4), (torch.zeros((2, 9), dtype=torch.int32)[:, 3:7], 9), (torch.zeros((6, 4), dtype=torch.int32)[::3], 12),
    (torch.zeros(8, dtype=torch.int32).unfold(0, 4, 4), 4), (torch.zeros((2, 4), dtype=torch.int32)[:, :0], 4),
])
def test_tables_that_are_parts_of_others(table, stride):
    pool = Tensor.empty_cache((6, 2, 16, 64), CPU)
    seqs = Sequences(2, ints(0, 3, 4), 3, ints(5, 6), table)
    for op in (pool.cache_write_paged(zeros(4, 128), seqs).op.desc, zeros(4, 512).attention_paged(pool, pool, seqs).op.desc.cache):
        assert (op.table_width, op.table_stride) == (table.shape[1], stride)


def test_one_sequence_has_a_row_of_any_stride():
    """There is no second row: a row that is repeated once, or a row of a transposed tensor."""
    pool = Tensor.empty_cache((6, 2, 16, 64), CPU)
    for table in (ints(0, 1, 2, 3)[None].expand(1, 4), torch.zeros((1, 4), dtype=torch.int32).as_strided((1, 4), (1, 1))):
        desc = zeros(4, 512).attention_paged(pool, pool, Sequences(1, ints(0, 4), 4, ints(5), table)).op.desc.cache
        assert (desc.table_width, desc.table_stride) == (4, 4)


@pytest.mark.parametrize("name,value", [("lens", ints(5)), ("starts", ints(0)), ("table", torch.zeros((1, 1), dtype=torch.int32)), ("batch", 9), ("max_rows", 4), ("max_keys", 64)])
def test_sequences_stay_as_they_were_made(name, value):
    """An operator checks the tensors when it is made and reads them when it runs: another, shorter one in between would be read past its end."""
    seqs = Sequences(2, ints(0, 3, 4), 3, ints(5, 6), torch.zeros((2, 4), dtype=torch.int32))
    kept = getattr(seqs, name)
    with pytest.raises(AttributeError):
        setattr(seqs, name, value)
    assert getattr(seqs, name) is kept
    seqs.lens.copy_(ints(7, 8))      # what they hold may change
    assert seqs.lens.tolist() == [7, 8]
