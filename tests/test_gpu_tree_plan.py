"""Tree drafting on the GPU, what lies between the four calls."""
import pytest
import torch

from tree_helpers import D, DEV

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
PARENTS = torch.tensor([[-1, 0, 0, 1, 1, 2]] * 2)


@pytest.fixture(scope="module")
def gqa(built_lib):
    import llminfer_b200 as pkg
    return pkg


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_plan_is_done_with_its_inputs_when_it_returns(gqa, kind):
    """A serving loop refills its pinned buffers for the next step while the stream is still busy."""
    tree = gqa.DraftTree(2, 6, 8, 2, DEV)
    parents, sizes, history = (t.to(kind).pin_memory() for t in (PARENTS, torch.tensor([6, 4]), torch.tensor([20, 30])))
    tree.plan(PARENTS)  # what a first call loads keeps it waiting for the stream
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)  # the stream is at work for some 50 ms
    tree.plan(parents, sizes, history)
    for t in (parents, sizes, history):
        t.zero_()
    torch.cuda.synchronize()
    mask, depth = gqa.tree_masks(PARENTS, torch.tensor([6, 4]))
    assert torch.equal(tree.parents.cpu(), PARENTS.int()) and tree.sizes.tolist() == [6, 4]
    assert tree.history.tolist() == [20, 30] and tree.lens.tolist() == [26, 34]
    assert torch.equal(tree.mask.cpu(), mask) and torch.equal(tree.depth.cpu(), depth)
