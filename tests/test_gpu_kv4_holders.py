"""A grow (madi_kv4_grow) of sequences whose last pages have other holders: sequences of the table, or
elsewhere (prompts kept for later requests).  Every array against the same steps on the host, whole numbers equal."""
import random

import numpy as np
import pytest

import pages_ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv4():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import madi_amd.kv4 as kv4
    import madi_amd.q8 as q8
    q8.init()
    return kv4


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


class Both:
    """The GPU's pages and the reference's."""

    def __init__(self, kv4, n_pages, page, b, max_pages, m):
        self.kv4, zeros = kv4, np.zeros
        self.ref = pages_ref.Pages(zeros(n_pages, np.int32), np.full((b, max_pages), -1, np.int32), zeros(b, np.int32), page)
        self.gpu = kv4.pages(n_pages, page, b, max_pages, m=m)

    def same(self):
        for name in ("lens", "refs", "table"):
            np.testing.assert_array_equal(getattr(self.gpu, name).cpu().numpy(), getattr(self.ref, name), err_msg=name)
        assert int(self.gpu.state[0]) == int((self.ref.refs == 0).sum())
        assert not self.gpu.mark[:len(self.ref.refs)].any()

    def hold(self, pages, n=1):
        """Held (or given back: n < 0) elsewhere; the number of free pages follows."""
        self.ref.refs[pages] += n
        self.gpu.refs.copy_(dev(self.ref.refs))
        self.gpu.state[0] = int((self.ref.refs == 0).sum())

    def grow(self, add, copy=None):
        add = np.asarray(add)
        self.kv4.kvGrow(self.gpu, dev(add)) if copy is None else self.kv4.kvGrow(self.gpu, dev(add), copy=copy)
        expect = self.ref.grow(add, self.gpu.m, copy)
        for name, e in zip(("row_off", "copies", "row_seq", "row_pos", "slot"), expect):
            if name != "copies" or copy is not False:
                np.testing.assert_array_equal(getattr(self.gpu, name).cpu().numpy(), e, err_msg=name)
        assert int(self.gpu.state[1]) == self.ref.left_out
        self.same()
        return expect[1]

    def trim(self, to):
        self.kv4.kvTrim(self.gpu, dev(to))
        self.ref.trim(np.asarray(to))
        self.same()

    def fork(self, parent, beams):
        self.kv4.kvFork(self.gpu, dev(parent), beams)
        self.ref.fork(np.asarray(parent), beams)
        self.same()


def test_a_page_held_elsewhere_is_appended_to(kv4):
    """By default; what another sequence has too is copied, held elsewhere or not; copy=True copies either."""
    t = Both(kv4, 40, 16, 6, 4, m=200)
    t.grow([5, 20, 16, 0, 7, 0])
    t.hold([0, 1, 2, 3, 4])
    assert (t.grow([1, 1, 1, 1, 1, 0]) == -1).all()
    t.fork([[0, 1, 2], [1, 1, 1]], 3)     # the fifth one's page has three sequences
    assert t.grow([1, 1, 0, 1, 1, 1])[:, 0].tolist() == [-1, -1, -1, 4, 4, 4]  # (and a holder elsewhere that does not grow)
    assert t.grow([1, 1, 0, 0, 0, 0], copy=True)[:, 0].tolist() == [0, 2, -1, -1, -1, -1]
    t.hold([0, 1, 2, 3, 4], -1)
    t.fork([[0, 0, 2], [0, 1, 2]], 3)
    assert (t.grow([0, 1, 0, 0, 0, 0])[:, 0] >= 0).tolist() == [False, True, False, False, False, False]


@pytest.mark.parametrize("groups,beams,max_pages,m", [(1, 1, 8, 40), (4, 5, 6, 60), (16, 4, 4, 64), (13, 5, 4, 100), (60, 17, 3, 1020),
                                                      (64, 16, 4, 20000), (65, 16, 4, 1040), (300, 7, 3, 2100), (300, 7, 3, 30000)])
def test_kept_prompts_and_beams(kv4, groups, beams, max_pages, m):
    """Sequences alone on pages that are held elsewhere, beams that share pages, both, in rows far apart: on either side
    of a wave's 64 sequences and a tile's 1024, through one workgroup and through the plan's launches."""
    rng = np.random.default_rng(groups + m)
    b, page = groups * beams, 16
    t = Both(kv4, b * max_pages + 9, page, b, max_pages, m=m)
    first = np.zeros(b, int)
    first[::beams] = rng.integers(1, 2 * page, groups)
    first[rng.integers(0, b, b // 8)] = 3
    while first.sum() > m:
        first[rng.integers(0, b, b // 8 + 1)] = 0
    t.grow(first)
    parent = np.where(rng.random((groups, beams)) < 0.4, 0, np.arange(beams))
    t.fork(parent, beams)
    # sequences of other groups begin with the first one's pages, as a host hands a kept prompt on
    for i in range(b - 1, b - 1 - b // 16, -1):
        if t.ref.lens[i] == 0:
            c = t.ref.count(int(t.ref.lens[0]))
            t.ref.lens[i], t.ref.table[i, :c] = t.ref.lens[0], t.ref.table[0, :c]
            t.ref.refs[t.ref.table[0, :c]] += 1
    t.gpu.lens.copy_(dev(t.ref.lens))
    t.gpu.table.copy_(dev(t.ref.table))
    used = np.flatnonzero(t.ref.refs)
    t.hold(used[rng.random(len(used)) < 0.5])
    for share in (1, 0.7, 0.5):
        t.grow((rng.random(b) < share) * rng.integers(1, 3))
        parent = np.where(rng.random((groups, beams)) < 0.3, rng.integers(0, beams, (groups, 1)), np.arange(beams))
        t.fork(parent, beams)
    t.grow((rng.random(b) < 0.6).astype(int), copy=True)


def contents(kv4, n_pages, page, b, max_pages, m):
    """Both with what the pages hold; the GPU's tables, copies and slots say where."""
    t, held = Both(kv4, n_pages, page, b, max_pages, m), pages_ref.Contents(n_pages, page, b)

    def take(name, arg, copy=None):
        arg = np.asarray(arg)
        if name == "grow":
            t.grow(arg, copy)
            held.grow(*(getattr(t.gpu, x).cpu().numpy() for x in ("copies", "row_seq", "slot")))
        else:
            for x in (t, held):
                x.fork(arg, arg.shape[1]) if name == "fork" else x.trim(arg)
        held.check(t.gpu.table.cpu().numpy(), t.gpu.lens.cpu().numpy())
    return t, take


@pytest.mark.parametrize("copy", [None, True])
@pytest.mark.parametrize("m", [9, 5000])
def test_a_sequence_that_is_left_out_keeps_its_tokens(kv4, m, copy):
    """The one that would copy finds no page, a shorter one asks for the page as well: the longer keeps it."""
    t, take = contents(kv4, 2, 16, 3, 2, m)
    for name, arg in (("grow", [5, 0, 0]), ("fork", [[0, 0, 0]]), ("grow", [1, 1, 1]), ("fork", [[0, 2, 1]]), ("grow", [0, 1, 1])):
        take(name, arg, copy)
    assert t.ref.lens.tolist() == [6, 7, 5] and t.ref.left_out == 1
    t, take = contents(kv4, 1, 16, 3, 2, m)
    for name, arg in (("grow", [6, 0, 0]), ("fork", [[0, 0, 0]]), ("trim", [9, 0, 3]), ("grow", [1, 0, 1])):
        take(name, arg, copy)
    assert t.ref.lens.tolist() == [7, 0, 3] and t.ref.left_out == 1


@pytest.mark.parametrize("groups,beams,page,share,m", [(1, 3, 16, 0.7, 9), (5, 4, 16, 0.7, 40), (5, 4, 32, 1.2, 4000), (60, 5, 16, 0.6, 500),
                                                       (60, 5, 16, 0.8, 9000), (275, 4, 16, 0.8, 2000), (275, 4, 64, 0.7, 15000)])
def test_holders_of_many_lengths(kv4, groups, beams, page, share, m):
    """Sequences cut down, forked and grown in any number, in pools that run short; one workgroup and the plan's."""
    rng = np.random.default_rng(groups * beams + m)
    b = groups * beams
    t, take = contents(kv4, int(b * share) + 1, page, b, 4, m)
    steps = pages_ref.holders_of_many_lengths(rng, b, beams, page, 4, m, 12 if b < 500 else 6)
    next(steps)
    while True:
        try:
            name, arg = steps.send(t.ref.lens)
        except StopIteration:
            break
        take(name, arg, None if rng.random() < 0.7 else True)


def test_pages_of_many_tokens(kv4):
    """Pages too large for a sequence's length and number to share a word: the longest keeps it, of equals the last."""
    for page in (1 << 16, 1 << 17, 1 << 20):
        n = page - 3
        t = Both(kv4, 8, page, 4, 2, m=page)
        t.grow([n, 0, 0, 0])
        t.fork([[0, 0, 0, 0]], 4)
        t.trim([n, n, n - 1, 5])
        assert (t.grow([1, 1, 1, 1])[:, 0] >= 0).tolist() == [True, False, True, True]
        t.fork([[1, 1, 1, 1]], 4)
        t.trim([n + 1, 1, 1 << 16 if page > 1 << 16 else 2, 1])
        assert (t.grow([0, 1, 1, 1])[:, 0] >= 0).tolist() == [False, True, True, True]
        t.trim([0, n, n, n])
        t.fork([[0, 2, 2, 2]], 4)
        assert (t.grow([0, 1, 1, 1])[:, 0] >= 0).tolist() == [False, True, True, False]


@pytest.mark.parametrize("b,m", [(150, 150), (20, 40), (1030, 1030), (150, 9000)])
def test_graph_replays_with_kept_prompts(kv4, b, m):
    """A captured grow, replayed after other pages were held, with eager steps between."""
    import madi_amd.q8 as q8
    rng = np.random.default_rng(b)
    t = Both(kv4, 3 * b, 16, b, 4, m)
    t.grow(np.minimum(rng.integers(1, 3, b), m // b))
    add = dev(np.ones(b))
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        q8.init(stream)
        kv4.kvGrow(t.gpu, add)
    q8.init()
    for k in range(4):
        used = np.flatnonzero(t.ref.refs)
        t.hold(used[rng.random(len(used)) < 0.4])
        if k % 2:
            t.fork(rng.integers(0, 2, (b // 2, 2)), 2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        expect = t.ref.grow(np.ones(b, int), m)
        t.same()
        for name, e in zip(("row_off", "copies", "row_seq", "row_pos", "slot"), expect):
            np.testing.assert_array_equal(getattr(t.gpu, name).cpu().numpy(), e, err_msg=name)
        t.grow((rng.random(b) < 0.5).astype(int))


@pytest.fixture
def cases():
    from perf import more_operators
    yield more_operators
    more_operators.own = False


def passes(cases, case, seed, own, n):
    cases.own = own
    st = cases.prepare(case, seed)
    return [[x.clone() for x in cases.run(st)] for _ in range(n)]


@pytest.mark.parametrize("draw", range(14))
def test_the_plain_form_of_growing_sequences(kv4, cases, draw):
    """The measured cases of page tables, in both forms; from the second pass on by what the first left."""
    listed = [c for c in cases.listed() if c["op"] in ("grow", "fork")]
    rng = random.Random(draw)
    case = listed[draw] if draw < len(listed) else next(c for c in iter(lambda: cases.draw(rng), None) if c["op"] == "grow")
    plain, here = (passes(cases, case, draw, own, 2) for own in (False, True))
    for p, h in zip(plain, here):
        for i, (x, y) in enumerate(zip(p, h)):
            assert torch.equal(x, y), (case, i)
