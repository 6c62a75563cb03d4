"""The policy operators at the ends of what they accept, against the plain implementations of
test_policy_gpu.py."""

import numpy as np
import pytest

from tests.test_policy_gpu import clean_status, dev, here, net  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,width", [(1, 2**31 - 4), (1, 2**31 - 1), (2, 2**30 - 1)])
def test_slot_rows_of_as_many_slots_as_there_may_be(net, rows, width):  # noqa: F811
    """A table of 2^31 - 1 slots or a little less: the column behind a row's last does not wrap around."""
    count, guard = 200, 64
    lengths = np.full(rows, count // rows, np.int32)
    entries, n = np.arange(7, 7 + count, dtype=np.int32), count // rows
    whole = torch.full((guard + rows * width + guard,), -6, dtype=torch.int32, device="cuda:0")
    table = whole[guard: guard + rows * width]  # 256 bytes in: its alignment is the buffer's
    starts = torch.full((rows + 1,), -5, dtype=torch.int32, device="cuda:0")
    where = torch.full((count,), -7, dtype=torch.int32, device="cuda:0")
    le, en = dev(lengths), dev(entries)
    net.slot_table(rows, width, le.data_ptr(), count, en.data_ptr(), starts.data_ptr(), table.data_ptr(),
                   where.data_ptr(), stream=here())
    torch.cuda.synchronize()
    assert (whole[:guard] == -6).all() and (whole[guard + rows * width:] == -6).all()
    assert starts.tolist() == [n * r for r in range(rows + 1)]
    for r in range(rows):
        row = table[r * width: (r + 1) * width]
        assert np.array_equal(row[:n].cpu().numpy(), entries[r * n: (r + 1) * n])
        assert int(row[n:].max()) == -1 == int(row[n:].min())
    assert np.array_equal(where.cpu().numpy(), np.concatenate([r * width + np.arange(n) for r in range(rows)]))
    assert net.status_word() == 0
