"""CPU checks of what the paged attention's Python entry hands to the library: CPU tensors stand for CUDA ones, and
the library's own checks of the arguments, which launch nothing, decide."""
import pytest
import torch

from kernelverse_b200 import _lib, ops

Q, CACHE, TABLE_STRIDE, BLOCK, MAX_LEN, WORKSPACE_BYTES = 0, 3, 14, 20, 22, -2      # places among the entry's arguments
WORKSPACE = 7                                                                       # the last check before the launch


@pytest.fixture
def attend(monkeypatch):
    """ops.paged_prefill_attention up to the launch: returns the arguments, or raises the library's refusal."""
    passed = []

    def call(name, *args):
        args = list(args)
        args[WORKSPACE_BYTES] = 0
        code = getattr(_lib.lib(), name)(*args)
        if code != WORKSPACE:
            raise _lib.KvbError(name, code, _lib.lib().kvb_last_error().decode())
        passed.append(args)

    monkeypatch.setattr(ops, "_device_of", lambda what, *ts: 0)
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(ops, "call", call)

    def run(**kw):
        a = dict(q=torch.zeros(4, 4, 64, dtype=torch.bfloat16), k_cache=torch.zeros(40, 16, 2, 64, dtype=torch.bfloat16),
                 v_cache=torch.zeros(40, 16, 2, 64, dtype=torch.bfloat16), qo_indptr=torch.tensor([0, 1, 4], dtype=torch.int32),
                 seq_lens=torch.tensor([20, 30], dtype=torch.int32), block_table=torch.zeros(2, 5, dtype=torch.int32))
        ops.paged_prefill_attention(**{**a, **kw})
        return passed[-1]

    return run


def test_the_places_of_the_arguments(attend):
    args = attend(max_seq_len=70)
    assert (args[TABLE_STRIDE], args[BLOCK], args[MAX_LEN]) == (5, 16, 70)
    assert attend()[MAX_LEN] == 80


@pytest.mark.parametrize("cut", [slice(3, 6), slice(0, 3), slice(5, 8)])
def test_lengths_past_a_column_slice_of_a_wider_table_are_refused(attend, cut):
    """A view's rows hold its columns, not those of the table that it was cut from: beyond them lie other entries, and
    behind the last row nothing."""
    table = torch.zeros(2, 8, dtype=torch.int32)[:, cut]
    args = attend(block_table=table, max_seq_len=48)
    assert args[TABLE_STRIDE] == 8 and args[MAX_LEN] == 48            # a view in place
    assert attend(block_table=table)[MAX_LEN] == 48
    for most in (49, 80, 128, 129):
        with pytest.raises(RuntimeError, match="max_seq_len"):
            attend(block_table=table, max_seq_len=most)


def test_lengths_past_other_views_are_refused(attend):
    for table in (torch.zeros(3, 2, dtype=torch.int32).t(), torch.zeros(1, 3, dtype=torch.int32).expand(2, 3),
                  torch.zeros(2, 6, dtype=torch.int32)[:, ::2]):
        assert attend(block_table=table, max_seq_len=48)[MAX_LEN] == 48
        with pytest.raises(RuntimeError, match="max_seq_len"):
            attend(block_table=table, max_seq_len=49)


@pytest.mark.parametrize("tokens", [1, 3])
def test_queries_off_the_16_byte_grid_are_copied(attend, tokens):
    """Rows of an odd width, one token's too (whose stride torch takes for contiguous), and a base between boundaries."""
    qo = torch.tensor([0, tokens, tokens], dtype=torch.int32)
    odd = torch.zeros(tokens * 259, dtype=torch.bfloat16).as_strided((tokens, 4, 64), (259, 64, 1))
    base = torch.zeros(tokens * 256 + 8, dtype=torch.bfloat16)
    at = next(i for i in range(8) if (base.data_ptr() + 2 * i) % 16 == 2)
    for q in (odd, base[at:at + tokens * 256].view(tokens, 4, 64)):
        args = attend(q=q, qo_indptr=qo)
        assert args[2] == 256 and args[Q] % 16 == 0 and args[Q] != q.data_ptr()
