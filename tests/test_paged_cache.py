"""paged.PagedCache and paged.AttentionPlan hold device addresses: what they describe can
neither be replaced behind the library's back nor be freed while a description of it lives."""

import pytest
import torch

from qgemv_b200 import paged


@pytest.mark.parametrize("kind,names", [
    (paged.PagedCache, ("k", "v", "table", "held", "page_size", "batch")),
    (paged.AttentionPlan, ("cache", "workspace", "held", "n_q_heads", "max_len", "weights")),
])
def test_descriptions_are_made_once(kind, names):
    made = object.__new__(kind)
    for name in names:
        setattr(made, name, 1)  # as the constructor does
        with pytest.raises(AttributeError, match=name):
            setattr(made, name, 2)
        assert getattr(made, name) == 1
    made.note = "a user's own"


@pytest.mark.gpu
def test_descriptions_keep_their_memory(cuda):
    mib = 1 << 20

    def used():
        return torch.cuda.memory_allocated()

    start = used()
    k, v = (torch.zeros(64, 8, 16, 128, dtype=torch.float16, device="cuda") for _ in range(2))  # 2 MiB each
    table = torch.zeros(1024, 256, dtype=torch.int32, device="cuda")                            # 1 MiB
    cache = paged.PagedCache(k, v, table)
    k.set_(torch.empty(0, dtype=torch.float16, device="cuda"))  # gives its storage up: the description keeps it
    held = cache.held
    del k, v, table, cache
    assert used() - start >= 5 * mib
    del held
    assert used() - start < mib

    cache = paged.PagedCache.empty(64, 8, 16, 128, 2, 4)
    plan = paged.AttentionPlan(cache, 16)
    space = plan.workspace.numel()
    held = plan.held
    del plan, cache
    assert used() - start >= space + 4 * mib
    del held
    assert used() - start < mib


@pytest.mark.gpu
def test_a_plan_outlives_the_names_of_its_cache(cuda):
    """The caller keeps the plan alone; nothing that it needs is handed out again."""
    k, v = (torch.randn(8, 2, 16, 64, device="cuda").half() for _ in range(2))
    cache = paged.PagedCache(k, v, torch.tensor([[5, 2]], dtype=torch.int32, device="cuda"))
    q, lens = torch.randn(1, 4, 64, device="cuda"), torch.tensor([20], dtype=torch.int32, device="cuda")
    plan = paged.AttentionPlan(cache, 4)
    want = paged.attend(plan, q, lens)
    with pytest.raises(AttributeError):
        cache.table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    plan.scale = 2 * plan.scale  # of the front end's own: may change
    assert not torch.equal(paged.attend(plan, q, lens), want)
    assert torch.equal(paged.attend(plan, q, lens, scale=plan.scale / 2), want)
    del cache, k, v
    refill = [torch.full((8, 2, 16, 64), float("nan"), device="cuda").half() for _ in range(4)]
    assert torch.equal(paged.attend(plan, q, lens, scale=plan.scale / 2), want) and len(refill) == 4
