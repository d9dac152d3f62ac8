"""Which form of the kernel a paged attention call takes, seen in the workspace that it asks for (on a GPU: SM counts)."""
import pytest
import torch


def _ctas(ops, tokens, sequences, group, dim, max_query):
    """(rows of a unit, CTAs) of the call: the workspace is CTAs * (32 + 2 * rows * (4 dim + 8)) bytes."""
    size = ops.paged_attention_workspace(tokens, sequences, 8 * group, 8, dim, 'cuda', max_query).numel()
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for rows, ctas in ((256, sms), (128, 2 * sms), (16, sms * {64: 4, 96: 3, 128: 2}[dim])):
        if size == ctas * (32 + 2 * rows * (4 * dim + 8)):
            return rows, ctas
    raise AssertionError(size)


@pytest.mark.gpu
@pytest.mark.parametrize('tokens,sequences,group,dim,max_query,rows', [
    (64, 64, 4, 128, 1, 16), (64, 16, 4, 128, 4, 16), (160, 32, 4, 128, 5, 128),          # single tokens, drafted ones
    (4096, 4, 4, 128, 1024, 256), (1000, 8, 1, 96, 125, 128), (1100, 8, 1, 96, 138, 256),  # chunks, of a tile at most and more
    (8447, 256, 4, 128, 8192, 128), (8200, 204, 4, 128, 2000, 128),                        # single tokens beside long chunks
    (10300, 100, 4, 128, 700, 256), (25500, 100, 4, 128, 2048, 256), (4030, 32, 8, 128, 2000, 256),
    (2942, 24, 6, 64, 626, 128), (4092, 24, 6, 64, 700, 256)])
def test_forms(tokens, sequences, group, dim, max_query, rows):
    from streamvoxel_b200 import ops
    assert _ctas(ops, tokens, sequences, group, dim, max_query)[0] == rows
