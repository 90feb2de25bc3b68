"""Forked requests and compaction: the manager's books, the scheduler's plans, and the step function on the CPU with the kernels
replaced by their plain statements."""
import random

import pytest
import torch

import kernel_refs
import plain_lfm2
from helpers import make_runner, rel_err
from neurogrid_b200.cache import CacheManager, OutOfPages, OutOfSlots, PagedNeed, PagePool
from neurogrid_b200.cache.storage import CacheStorage, page_bytes, parse_cache_dtype
from neurogrid_b200.cache.manager import SlotNeed
from neurogrid_b200.engine import Request, Scheduler, StepEntry
from neurogrid_b200.sampling import SamplingParams
from tiny_configs import PAGE_SIZE


def mgr(pages=(16,), page_size=8, max_requests=4, max_seq_len=256, windows=(None,)):
    return CacheManager([PagedNeed(2, 16, w) for w in windows], list(pages), page_size, max_requests, max_seq_len)


def test_pool_counts_holders():
    p = PagePool(3)
    a = p.take(1)[0]
    p.share(a)
    p.give_back(a)
    assert p.free == 2 and p.holders(a) == 1
    p.give_back(a)
    assert p.free == 3
    with pytest.raises(RuntimeError):
        p.give_back(a)
    with pytest.raises(ValueError):
        p.share(a)
    with pytest.raises(ValueError):
        p.share(9)


def test_fork_shares_full_pages_and_copies_the_last():
    m = mgr(pages=(6, 6), windows=(None, None))
    m.admit("a")
    m.extend("a", 19); m.advance("a", 19)                      # two full pages and three tokens
    src, dst, copies = m.fork("a", "b")
    assert src == m.slot("a") and dst == m.slot("b") and m.length("b") == 19
    for g in range(2):
        ta, tb = m.table("a", g), m.table("b", g)
        assert ta[:2] == tb[:2] and ta[2] != tb[2] and copies[g] == [(ta[2], tb[2])]
        assert m.pools[g].free == 2
    m.check()
    m.extend("b", 6); m.advance("b", 6)
    m.check()
    m.release("a")
    m.check()
    assert m.pages_free() == [2, 2]
    m.release("b")
    assert m.pages_free() == [6, 6]
    # a request that ends on a page's end shares everything
    m.admit("c")
    m.extend("c", 16); m.advance("c", 16)
    assert m.fork("c", "d")[2] == [[], []] and m.pages_free() == [4, 4]
    m.check()


def test_pages_that_a_fork_still_holds_are_not_counted_on():
    m = mgr(pages=(4,), windows=(8,), page_size=8)
    m.admit("a")
    m.extend("a", 24); m.advance("a", 24)                      # three pages, of which the window has passed two
    m.fork("a", "b")
    assert m.pages_free() == [1] and m.pages_freed_first("a") == [0]
    assert m.can_extend("a", 8) and not m.can_extend("a", 9)   # (a page is free; giving back two that b holds frees none)
    m.extend("a", 8); m.advance("a", 8)
    m.check()
    assert m.pages_free() == [0] and m.pages_freed_first("b") == [2] and m.can_extend("b", 9)
    m.extend("b", 9); m.advance("b", 9)
    m.check()


def test_fork_is_all_or_nothing():
    m = mgr(pages=(4, 3), windows=(None, None), max_requests=3)
    m.admit("a")
    m.extend("a", 17); m.advance("a", 17)
    assert not m.can_fork("a")
    with pytest.raises(OutOfPages):
        m.fork("a", "b")                                       # group 1 has no page left: group 0 must not be touched
    assert m.pages_free() == [1, 0] and m.slots_free() == 2 and not m.is_live("b")
    m.check()
    n = mgr(max_requests=1)
    n.admit("a")
    with pytest.raises(OutOfSlots):
        n.fork("a", "b")
    with pytest.raises(KeyError):
        n.fork("a", "a")


@pytest.mark.parametrize("seed", range(4))
def test_random_forks_and_compactions_keep_the_books_and_the_contents(seed):
    """Pages hold the token positions written to them; forks and compactions move contents as they say; every request still finds its own."""
    rng = random.Random(seed)
    ps = 4
    m = mgr(pages=(40, 30), page_size=ps, max_requests=6, windows=(None, 9), max_seq_len=80)
    store = [{}, {}]                                           # per group: page -> {place: (owner's mark, position)}
    marks, live, nxt = {}, [], 0

    def write(r, n):
        start = m.length(r)
        m.extend(r, n)
        for g in range(2):
            for pos in range(start, start + n):
                page = m.table(r, g)[pos // ps]
                if page >= 0:
                    assert m.pools[g].holders(page) == 1, "a shared page is written"
                    store[g].setdefault(page, {})[pos % ps] = marks[r][pos] if pos < len(marks[r]) else None
        m.advance(r, n)

    for step in range(400):
        op = rng.random()
        if op < 0.15 and len(live) < 6:
            m.admit(nxt); live.append(nxt); marks[nxt] = []; nxt += 1
        elif op < 0.6 and live:
            r = rng.choice(live)
            n = rng.choice([1, 1, 2, 5, 9])
            if m.can_extend(r, n):
                marks[r] += [(r, step, i) for i in range(n)]
                write(r, n)
        elif op < 0.75 and live and m.can_fork(live[0]):
            r = rng.choice(live)
            if m.can_fork(r):
                _, _, copies = m.fork(r, nxt)
                for g, pairs in enumerate(copies):
                    for a, b in pairs:
                        store[g][b] = dict(store[g].get(a, {}))
                marks[nxt] = list(marks[r]); live.append(nxt); nxt += 1
        elif op < 0.85:
            for g, moves in enumerate(m.compact()):
                assert not set(moves) & set(moves.values())
                for a, b in moves.items():
                    store[g][b] = dict(store[g].get(a, {}))
                held = m.pools[g].held_pages()
                assert held == list(range(len(held)))
        elif live:
            r = live.pop(rng.randrange(len(live)))
            m.release(r)
        m.check()
        for r in live:
            for g in range(2):
                lo = max(0, m.length(r) - 9 + 1) if g else 0
                for pos in range(lo, m.length(r)):
                    assert store[g][m.table(r, g)[pos // ps]][pos % ps] == marks[r][pos]


def test_scheduler_reads_a_prompt_once_and_forks_its_samples():
    m = mgr(pages=(32,), max_requests=4, max_seq_len=64)
    s = Scheduler(m, max_tokens_per_step=16, max_requests=4, chunk_size=16)
    params = SamplingParams(max_new_tokens=3)
    reqs = [Request(i, list(range(20)), params) for i in range(3)]
    s.add_samples(reqs[0], reqs[1:])
    fed, forks = 0, 0
    while s.has_work():
        plan = s.plan()
        forks += len(plan.forks)
        for e in plan.entries:
            if not m.is_live(e.request.id):
                m.admit(e.request.id)
            m.extend(e.request.id, e.count); m.advance(e.request.id, e.count)
            fed += e.count
        s.commit(plan, [7] * sum(e.sample for e in plan.entries))
        m.check()
    assert forks == 2 and [r.output for r in reqs] == [[7] * 3] * 3
    assert fed == 19 + 3 + 3 * 2                              # the prompt's last token and two of its own for each
    assert m.pages_free() == [32]


def test_samples_that_find_no_slot_read_the_prompt_themselves():
    m = mgr(pages=(32,), max_requests=2, max_seq_len=64)
    s = Scheduler(m, max_tokens_per_step=64, max_requests=2)
    reqs = [Request(i, list(range(9)), SamplingParams(max_new_tokens=2)) for i in range(4)]
    s.add_samples(reqs[0], reqs[1:])
    one = Request("one", [5], SamplingParams(max_new_tokens=2))
    s.add_samples(one, [Request("two", [5], SamplingParams(max_new_tokens=2))])
    while s.has_work():
        plan = s.plan()
        for e in plan.entries:
            if not m.is_live(e.request.id):
                m.admit(e.request.id)
            m.extend(e.request.id, e.count); m.advance(e.request.id, e.count)
        s.commit(plan, [1] * sum(e.sample for e in plan.entries))
        m.check()
    assert all(r.output == [1, 1] for r in reqs + [one])
    # a prompt that cannot be served fails with its samples
    t = Scheduler(mgr(pages=(1,)), max_tokens_per_step=64, max_requests=2)
    bad = [Request(i, list(range(30)), SamplingParams()) for i in range(2)]
    t.add_samples(bad[0], bad[1:])
    assert t.plan().failed == bad and all(r.finish_reason == "cache_full" for r in bad) and not t.has_work()


def copy_pages(pools, src, dst):
    for p in pools:
        p[:, list(dst)] = p[:, list(src)]


@pytest.mark.parametrize("name", ["A", "B", "D"])
def test_a_forked_request_goes_on_as_its_own(model_dirs, monkeypatch, name):
    kernel_refs.install(monkeypatch)
    monkeypatch.setattr("neurogrid_b200.csrc.ops.copy_pages", copy_pages)
    cfg, w = plain_lfm2.load_plain(model_dirs[name])
    g = torch.Generator().manual_seed(3)
    seq = torch.randint(0, cfg["vocab_size"], (45,), generator=g).tolist()
    other = seq[:37] + torch.randint(0, cfg["vocab_size"], (8,), generator=g).tolist()
    runner = make_runner(model_dirs[name], page_size=PAGE_SIZE[name], max_requests=4)
    runner.step([StepEntry("x", seq[:11])])                    # a neighbour that ends later: its pages leave gaps
    runner.step([StepEntry("a", seq[:37])])
    runner.fork("a", "b")
    runner.cache.check()
    got = {"a": [], "b": []}
    for i in range(37, 45):
        if i == 40:
            runner.finish("x")
            runner.compact()
            runner.cache.check()
        out = runner.step([StepEntry("a", [seq[i]], [0]), StepEntry("b", [other[i]], [0])])
        got["a"].append(out[0].clone()); got["b"].append(out[1].clone())
    for r, tokens in (("a", seq), ("b", other)):
        assert rel_err(torch.stack(got[r]), plain_lfm2.forward(cfg, w, tokens)[37:]) < 2e-5
    held = runner.cache.pools[0].held_pages()
    assert set(held) <= set(range(len(held) + 2))              # (pages taken after the compaction may lie behind a gap's end)


def test_storage_in_8_bits():
    needs = {0: PagedNeed(2, 32, eight_bit=True), 1: PagedNeed(2, 32, eight_bit=True), 2: PagedNeed(1, 24, 9), 3: SlotNeed((2, 3))}
    st = CacheStorage(needs, pages_per_group=6, page_size=32, max_requests=3, dtype=torch.bfloat16, device="cpu", cache_dtype=torch.int8)
    assert st.k[0].dtype == st.v[0].dtype == torch.int8 and st.k[0].shape == (2, 6, 2, 32, 32)
    assert st.k_scales[0].shape == (2, 6, 2, 2) and st.k_scales[0].dtype == torch.float32
    assert st.k[1].dtype == torch.bfloat16 and st.k_scales[1] is None
    assert [len(st.pools(g)) for g in range(2)] == [4, 2]
    per_page = page_bytes(needs[0], 32, torch.bfloat16, torch.int8)
    assert per_page == 2 * 2 * 32 * 32 + 2 * 2 * 2 * 4 and page_bytes(needs[2], 32, torch.bfloat16, torch.int8) == 2 * 24 * 32 * 2
    assert sum(t[0, 0].numel() * t.element_size() for t in st.pools(0)) == per_page
    assert st.nbytes() == sum(t.numel() * t.element_size() for g in range(2) for t in st.pools(g)) + st.state[0].numel() * 4
    small = CacheStorage({0: needs[0]}, pages_per_group=2, page_size=8, max_requests=1, dtype=torch.bfloat16, device="cpu",
                         cache_dtype=torch.float8_e4m3fn)
    assert small.k_scales[0].shape == (1, 2, 2, 1)
    with pytest.raises(ValueError, match="at least 8"):
        CacheStorage(needs, pages_per_group=2, page_size=4, max_requests=1, dtype=torch.bfloat16, device="cpu", cache_dtype=torch.int8)
    assert parse_cache_dtype("e4m3") == torch.float8_e4m3fn and parse_cache_dtype(None) is None
    with pytest.raises(ValueError, match="unknown cache type"):
        parse_cache_dtype("fp4")


def test_a_model_that_cannot_hold_its_cache_in_8_bits_says_so(model_dirs, metanex_dirs):
    from neurogrid_b200.engine import ModelRunner
    from neurogrid_b200.engine.loading import model_from_dir
    _, f32 = model_from_dir(model_dirs["A"], dtype="float32", device="cpu")
    with pytest.raises(ValueError, match="bfloat16"):
        ModelRunner(f32, num_pages=4, cache_dtype="e4m3")
    _, other = model_from_dir(sorted(metanex_dirs.values())[0], dtype="bfloat16", device="cpu")
    with pytest.raises(ValueError, match="no layer"):
        ModelRunner(other, num_pages=4, cache_dtype="int8")
