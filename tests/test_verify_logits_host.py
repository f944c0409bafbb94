"""SpeculativeTree.verify_logits without a GPU: what it asks of its context."""
import numpy as np
import pytest

import velokv
from velokv import branching_tree


class Buffer:
    def __init__(self, nbytes, ptr):
        self.nbytes, self.ptr, self.data = nbytes, ptr, np.zeros(nbytes, np.uint8)

    def download(self, shape=None, dtype=None, offset=0):
        n = int(np.prod(shape)) * np.dtype(dtype).itemsize
        assert 0 <= offset <= offset + n <= self.nbytes
        return self.data[offset:offset + n].view(dtype).reshape(shape)


class FakeContext:
    """Records the call and answers node i with token 10 i and log probability -i / 2, at the addresses given."""

    def __init__(self, scratch):
        self.scratch, self.buffers, self.calls = scratch, [], []

    def alloc(self, nbytes):
        self.buffers.append(Buffer(nbytes, 1 << 20 << len(self.buffers)))
        return self.buffers[-1]

    def token_logprobs_workspace_bytes(self, n_rows, vocab, n_top=0, dtype=velokv.DT_F16):
        assert n_top == 1
        return self.scratch

    def span(self, at, nbytes):
        """The buffer bytes that an address (or a buffer) names."""
        at = getattr(at, "ptr", at)
        b = next(b for b in self.buffers if b.ptr <= at and at + nbytes <= b.ptr + b.nbytes)
        return b.data[at - b.ptr:at - b.ptr + nbytes], (at, at + nbytes)

    def token_logprobs(self, logits, dtype, n_rows, vocab, top_ids=None, top_logprobs=None, n_top=0, row_stride=0,
                       workspace=None, workspace_bytes=0, stream=None):
        ids, a = self.span(top_ids, 4 * n_rows)
        top, b = self.span(top_logprobs, 4 * n_rows)
        spans = [a, b] + ([self.span(workspace, workspace_bytes)[1]] if workspace_bytes else [])
        spans.sort()
        assert all(x[1] <= y[0] for x, y in zip(spans, spans[1:]))  # nothing overlaps
        ids[:] = np.arange(0, 10 * n_rows, 10, dtype=np.int32).view(np.uint8)
        top[:] = (-np.arange(n_rows) / 2).astype(np.float32).view(np.uint8)
        self.calls.append((workspace, workspace_bytes, stream))

    def sync(self, stream=None):
        assert stream == self.calls[-1][2]


@pytest.mark.parametrize("n_nodes", [1, 7, 32])
@pytest.mark.parametrize("scratch", [0, 4, 1000])
def test_scratch_is_the_calls_own(n_nodes, scratch):
    """Two trees verified at once on two streams share nothing: the context's scratch is not used."""
    tree, ctx = branching_tree([2, 2, 2, 2, 2], n_nodes), FakeContext(scratch)
    got = tree.verify_logits(ctx, 4096, velokv.DT_F16, 32000, stream="a stream")
    workspace, nbytes, _ = ctx.calls[0]
    assert nbytes >= scratch and (not scratch or (getattr(workspace, "ptr", workspace) or 0) % 16 == 0)
    assert scratch == 0 or workspace is not None
    assert got.expected == list(range(0, 10 * n_nodes, 10)) and got.logprobs == [-i / 2 for i in range(n_nodes)]
