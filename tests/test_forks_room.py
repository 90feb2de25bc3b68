"""Forked samples in a pool with little room: the headroom that admissions leave, and copies of forks that are preempted at once."""
import pytest

from neurogrid_b200.cache import CacheManager, PagedNeed
from neurogrid_b200.engine import Request, Scheduler
from neurogrid_b200.sampling import SamplingParams


def mgr(pages, page_size=8, max_requests=4, max_seq_len=256):
    return CacheManager([PagedNeed(2, 16, None)], [pages], page_size, max_requests, max_seq_len)


def run(s, m, plan):
    fed = 0
    for e in plan.entries:
        if not m.is_live(e.request.id):
            m.admit(e.request.id)
        m.extend(e.request.id, e.count); m.advance(e.request.id, e.count)
        fed += e.count
    s.commit(plan, [7] * sum(e.sample for e in plan.entries))
    m.check()
    return fed


@pytest.mark.parametrize("tokens", [17, 20])                   # all but the last: whole pages, or a page begun
@pytest.mark.parametrize("pages", range(4, 12))
def test_samples_are_forked_only_where_every_running_request_keeps_a_page(tokens, pages):
    """No fork is preempted in the plan that makes it, and what is forked goes on without reading the prompt again."""
    m = mgr(pages)
    s = Scheduler(m, max_tokens_per_step=64, max_requests=4)
    reqs = [Request(i, list(range(tokens)), SamplingParams(max_new_tokens=3)) for i in range(4)]
    s.add_samples(reqs[0], reqs[1:])
    fed = forks = 0
    for _ in range(200):
        if not s.has_work():
            break
        plan = s.plan()
        forks += len(plan.forks)
        assert not plan.failed and not plan.preempted
        fed += run(s, m, plan)
    assert [r.output for r in reqs] == [[7] * 3] * 4 and all(r.preemptions == 0 for r in reqs)
    assert fed == 4 * 3 + (4 - forks) * (tokens - 1) and m.pages_free() == [pages]
    free, running = pages - -(-(tokens - 1) // 8), 1
    while running < 4 and free > running:
        free, running = free - (1 if tokens == 20 else 0), running + 1
    assert forks == running - 1


def test_copies_of_a_fork_that_is_preempted_in_its_plan_are_not_made():
    """An older request takes the pages that were there when the fork was made."""
    m = mgr(7)
    s = Scheduler(m, max_tokens_per_step=64, max_requests=4)
    params = SamplingParams(max_new_tokens=4)
    old, parent, fork = Request("old", list(range(48)), params), Request("parent", list(range(9)), params), Request("fork", list(range(9)), params)
    for r, fed in ((old, 24), (parent, 8)):
        s.add(r)
        s.waiting.remove(r)
        m.admit(r.id); m.extend(r.id, fed); m.advance(r.id, fed)
        r.fed, r.state = fed, "running"
        s.running.append(r)
    fork.key, parent.forks = 5, [fork]
    plan = s.plan()
    assert fork in plan.preempted and plan.forks == [] and not m.is_live("fork")
    assert [e.request for e in plan.entries] == [old]
    run(s, m, plan)
