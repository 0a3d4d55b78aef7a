"""Arguments of tree_verify beside its tensors: calls without a workspace."""
import pytest
import torch

from frisk_amd import runtime as rt
from tests.gpu_util import randn

pytestmark = pytest.mark.gpu


def args(batch, tokens, vocab):
    i32 = dict(dtype=torch.int32, device="cuda")
    parents = torch.arange(-1, tokens - 1, **i32).expand(batch, tokens).contiguous()
    return (randn((batch, tokens, vocab), vocab), torch.zeros(batch, tokens, **i32), parents,
            torch.full((batch, tokens), 0.5, device="cuda"), torch.full((batch,), 0.5, device="cuda"))


@pytest.mark.parametrize("workspace", [False, None])
def test_without_a_workspace(workspace):
    # One node of a short row takes none.
    one = args(3, 1, 500)
    assert rt.tree_verify_workspace_bytes(3, 1, 500, torch.float32) == 0
    want = rt.tree_verify(*one)
    got = rt.tree_verify(*one, workspace=workspace)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # Trees do.
    need = rt.tree_verify_workspace_bytes(3, 4, 500, torch.float32)
    assert need > 0
    with pytest.raises(ValueError, match=f"workspace of 0 bytes, this call takes {need}"):
        rt.tree_verify(*args(3, 4, 500), workspace=workspace)


def test_a_workspace_of_the_caller():
    need = rt.tree_verify_workspace_bytes(3, 4, 500, torch.float32)
    want = rt.tree_verify(*args(3, 4, 500))
    got = rt.tree_verify(*args(3, 4, 500), workspace=torch.empty(need, dtype=torch.uint8, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for short in (torch.empty(need - 1, dtype=torch.uint8, device="cuda"),
                  torch.empty(need, dtype=torch.uint8), torch.empty(2 * need, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ValueError, match="workspace"):
            rt.tree_verify(*args(3, 4, 500), workspace=short)
