"""GPU page operations (grow, fork, free, compact) against the sequential oracle, exact; and a serving run of them
with append and attention."""

import numpy as np
import pytest
import torch

from oracle import fp4 as of

pytestmark = pytest.mark.gpu


def _ia():
    import intent_attention
    return intent_attention


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _state(seed, P, PS, S, Ht, W, lengths, share=0.2, D=64):
    """A pool of fp16 pages and slots that hold random pages, some of them shared."""
    ia = _ia()
    g = np.random.default_rng(seed)
    refs = np.zeros(P, np.int32)
    table = np.full((S, Ht, W), -1, np.int32)
    order = list(g.permutation(P))
    given = []
    for s in range(S):
        for h in range(Ht):
            for w in range(-(-lengths[s] // PS)):
                if given and g.random() < share:
                    p = given[g.integers(len(given))]
                else:
                    p = order.pop()
                    given.append(p)
                table[s, h, w] = p
                refs[p] += 1
    k, v = (g.standard_normal((P, PS, D)).astype(np.float16) for _ in range(2))
    pool = ia.PagePool(P, PS, D, k_f16=torch.from_numpy(k).cuda(), v_f16=torch.from_numpy(v).cuda())
    pages = ia.SequencePages(_i32(refs), _i32(table), _i32(lengths), PS)
    return pool, pages, of.Pages(refs, table, np.asarray(lengths, np.int32), PS, (k, v))


def _same(pool, pages, want, data=True):
    np.testing.assert_array_equal(pages.lengths.cpu().numpy(), want.lengths)
    np.testing.assert_array_equal(pages.table.cpu().numpy(), want.table)
    np.testing.assert_array_equal(pages.refs.cpu().numpy(), want.refs)
    if data:
        np.testing.assert_array_equal(pool.k_f16.cpu().numpy(), want.planes[0])
        np.testing.assert_array_equal(pool.v_f16.cpu().numpy(), want.planes[1])


def _counter():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("P,PS,S,Ht,W", [(64, 16, 4, 1, 6), (5000, 16, 33, 4, 9), (20000, 8, 64, 8, 12),
                                         (9001, 3, 700, 2, 5), (1, 16, 1, 1, 1)])
def test_grow(P, PS, S, Ht, W):
    g = np.random.default_rng(P)
    lengths = g.integers(0, W * PS // 2 + 1, S).tolist() if P > 1 else [0]
    pool, pages, want = _state(P, P, PS, S, Ht, W, lengths)
    more = g.integers(0, W * PS // 2 + 1, S)
    more[g.random(S) < 0.3] = 0
    more[-1] = 1
    if S > 3:
        more[1], more[2] = -4, W * PS + 1
    r = _counter()
    _ia().grow_sequences(pool, pages, _i32(more), rejected=r)
    want.grow(more)
    _same(pool, pages, want)
    assert int(r) == want.rejected


@pytest.mark.parametrize("S,Ht,P", [(1100, 9, 40000), (260, 17, 9000), (5000, 1, 12000)])
def test_grow_many_rows(S, Ht, P):
    """More rows than a block plans at a time, and free pages that end among the slots."""
    g = np.random.default_rng(S)
    W, PS = 4, 4
    lengths = g.integers(0, W * PS // 2 + 1, S).tolist()
    pool, pages, want = _state(S, P, PS, S, Ht, W, lengths, share=0.3, D=8)
    r = _counter()
    for _ in range(2):
        more = g.integers(0, W * PS // 2, S)
        more[g.random(S) < 0.4] = 0
        _ia().grow_sequences(pool, pages, _i32(more), rejected=r)
        want.grow(more)
        _same(pool, pages, want)
        assert int(r) == want.rejected
    assert want.rejected > 0


@pytest.mark.parametrize("PS,D", [(256, 128), (100, 128), (1000, 24), (129, 100)])
def test_pages_of_several_pieces(PS, D):
    """Pages that several warps copy, with ends inside a piece, by grow and by compact."""
    S, W = 6, 3
    pool, pages, want = _state(PS, 60, PS, S, 2, W, [PS + 3, 2 * PS, 5, 0, PS - 1, 2 * PS + 9], share=0.6, D=D)
    more = [1, 1, PS, 2, 3, 0]
    _ia().grow_sequences(pool, pages, _i32(more))
    want.grow(more)
    _same(pool, pages, want)
    _ia().free_sequences(pages, _i32([0, 3]))
    want.free([0, 3])
    assert int(_ia().compact_pages(pool, pages)) == want.compact()
    _same(pool, pages, want)


def test_grow_runs_out():
    """Everything up to the first slot that does not fit; later ones stay, those without tokens too."""
    pool, pages, want = _state(3, 40, 16, 6, 2, 8, [17, 5, 0, 40, 16, 3], share=0.5)
    more = [16, 30, 60, 16, 1, 0]
    r = _counter()
    _ia().grow_sequences(pool, pages, _i32(more), rejected=r)
    want.grow(more)
    _same(pool, pages, want)
    assert int(r) == want.rejected
    more = [100, 1, 90, 1, 100, 13]
    _ia().grow_sequences(pool, pages, _i32(more), rejected=r)
    want.grow(more)
    _same(pool, pages, want)
    assert int(r) == want.rejected > 0


def test_grow_refuses_a_missing_open_page():
    pool, pages, want = _state(5, 64, 16, 3, 2, 4, [20, 16, 5], share=0.0)
    for t in (pages.table, ):
        t[0, 1, 1] = -1
    want.table[0, 1, 1] = -1
    r = _counter()
    _ia().grow_sequences(pool, pages, _i32([1, 1, 1]), rejected=r)
    want.grow([1, 1, 1])
    _same(pool, pages, want)
    assert int(r) == want.rejected == 1


@pytest.mark.parametrize("S,Ht,W", [(8, 1, 3), (24, 8, 40), (64, 3, 300)])
def test_fork_and_free(S, Ht, W):
    g = np.random.default_rng(S)
    PS = 16
    lengths = [int(g.integers(0, W * PS + 1)) if s < S // 2 else 0 for s in range(S)]
    pool, pages, want = _state(S, S * Ht * W + 5, PS, S, Ht, W, lengths)
    src = g.integers(0, S // 2, S // 2 + 3)
    dst = np.concatenate([g.permutation(np.arange(S // 2, S))[:S // 2 - 1], [0, S, S // 2, -1]])
    r = _counter()
    _ia().fork_sequences(pages, _i32(src), _i32(dst), rejected=r)
    want.fork(list(src), list(dst))
    _same(pool, pages, want)
    assert int(r) == want.rejected > 0
    slots = list(g.permutation(S)[:S // 2 + 1]) + [S + 1, -1]
    slots += slots[:2]
    _ia().free_sequences(pages, _i32(slots), rejected=r)
    want.free(slots)
    _same(pool, pages, want)
    assert int(r) == want.rejected
    _ia().free_sequences(pages, _i32(list(range(S))))
    assert int(pages.refs.abs().max()) == 0 and int((pages.table >= 0).sum()) == 0


def test_fork_of_a_destination_is_refused():
    pool, pages, want = _state(7, 64, 16, 4, 1, 4, [40, 0, 0, 0])
    r = _counter()
    _ia().fork_sequences(pages, _i32([0, 1, 2, 3]), _i32([1, 2, 2, 3]), rejected=r)
    want.fork([0, 1, 2, 3], [1, 2, 2, 3])
    _same(pool, pages, want)
    assert int(r) == want.rejected == 3
    assert pages.lengths.tolist() == [40, 40, 0, 0]


@pytest.mark.parametrize("S,Ht,W", [(5, 1, 3), (40, 8, 30)])
def test_shrink(S, Ht, W):
    """Draft tokens given back: pages without a token go, shared ones count down, and growing again copies an open
    page that others hold."""
    g = np.random.default_rng(S)
    lengths = g.integers(0, W * 16 + 1, S).tolist()
    pool, pages, want = _state(S, 4 * S * Ht * W + 5, 16, S, Ht, W, lengths, share=0.4)
    off = np.minimum(g.integers(0, W * 16, S), lengths)
    off[0], off[1], off[2] = lengths[0], lengths[1] + 1, -1
    r = _counter()
    _ia().shrink_sequences(pages, _i32(off), rejected=r)
    want.shrink(off)
    _same(pool, pages, want)
    assert int(r) == want.rejected == 2 and int(pages.lengths[0]) == 0
    more = g.integers(0, 3, S)
    _ia().grow_sequences(pool, pages, _i32(more), rejected=r)
    want.grow(more)
    _same(pool, pages, want)
    assert int(r) == want.rejected


@pytest.mark.parametrize("P,S,Ht,W", [(64, 3, 1, 4), (8192, 16, 4, 20), (70001, 32, 8, 100), (1, 1, 1, 1)])
def test_compact(P, S, Ht, W):
    g = np.random.default_rng(P)
    lengths = g.integers(0, W * 16 + 1, S).tolist()
    pool, pages, want = _state(P + 1, P, 16, S, Ht, W, lengths, share=0.3)
    n = _ia().compact_pages(pool, pages)
    assert int(n) == want.compact()
    _same(pool, pages, want)
    assert bool((pages.refs[:int(n)] > 0).all()) and not bool(pages.refs[int(n):].any())
    assert int(_ia().compact_pages(pool, pages)) == want.compact()      # nothing left to move
    _same(pool, pages, want)


def test_tagged_pages_copy_their_format():
    """Only the planes of a page's format move, with its tag; odd plane sizes included."""
    ia = _ia()
    P, PS, D = 40, 16, 64
    pool = ia.PagePool.allocate(P, PS, D, scale_mode="page", zero=True)
    g = np.random.default_rng(0)
    fmts = g.integers(1, 6, P).astype(np.uint8)
    pool.quantize_(torch.randn(P, PS, D, device="cuda"), torch.randn(P, PS, D, device="cuda"),
                   torch.from_numpy(fmts).cuda())
    from intent_attention.paged import make_tag_map
    tag_map = make_tag_map({c: c for c in range(6)})
    for dtype in (torch.uint8, torch.int32):
        before = {n: getattr(pool, n).clone() for n in vars(pool) if torch.is_tensor(getattr(pool, n))}
        tags = torch.from_numpy(fmts).cuda().to(dtype)
        ids = g.permutation(P)[:9]
        refs = np.zeros(P, np.int32)
        refs[ids] = 1
        pages = ia.SequencePages(_i32(refs), _i32(ids.reshape(1, 1, 9)), _i32([9 * PS]), PS)
        ia.compact_pages(pool, pages, page_tags=tags, tag_map=tag_map)
        new = pages.table.cpu().numpy().ravel()
        for a, b in zip(ids, new):
            assert int(tags[b]) == fmts[a]
            names = {1: ["f16"], 2: ["fp8", "scale"], 3: ["i8", "scale"], 4: ["i4", "scale"],
                     5: ["i4", "i4r", "scale", "res_scale"]}[int(fmts[a])]
            for n in names:
                for side in "kv":
                    assert torch.equal(getattr(pool, f"{side}_{n}")[b], before[f"{side}_{n}"][a])
        for n, t in before.items():
            getattr(pool, n).copy_(t)


PLANES = {0: [], 1: ["f16"], 2: ["fp8", "scale"], 3: ["i8", "scale"], 4: ["i4", "scale"],
          5: ["i4", "i4r", "scale", "res_scale"], 6: []}


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int32])
@pytest.mark.parametrize("op", ["grow", "compact"])
def test_tagged_pages_copy_nothing_else(op, dtype):
    """A page of every format (SKIP, SPARSE and a tag beyond the map included), by copy-on-write and by packing: the
    planes of its format and its tag arrive, every other byte of the pool stays."""
    ia = _ia()
    from intent_attention.paged import make_tag_map
    g = np.random.default_rng(3)
    P, PS, D = 48, 16, 64
    pool = ia.PagePool.allocate(P, PS, D, scale_mode="group32", zero=True)
    planes = {n: t for n, t in vars(pool).items() if torch.is_tensor(t)}
    assert len(planes) == 14
    for t in planes.values():
        t.view(torch.uint8).copy_(torch.from_numpy(g.integers(0, 255, (*t.shape[:-1], t.shape[-1] * t.element_size()),
                                                              dtype=np.uint8)))
    before = {n: t.view(torch.uint8).clone() for n, t in planes.items()}
    # tag 10 + format, 9 SPARSE; 200 is beyond the map: the default, INT8 as tag 3
    formats = [0, 1, 2, 3, 4, 5, 6, 3, 3]
    tag_of = [10, 11, 12, 13, 14, 15, 9, 3, 200]
    tag_map = make_tag_map({**{10 + c: c for c in range(6)}, 9: 6, 3: 3})
    tags = torch.full((P,), 11, dtype=dtype, device="cuda")
    S = len(formats)
    ids = 20 + g.permutation(P - 20)[:S]
    tags[torch.from_numpy(ids).cuda()] = torch.tensor(tag_of, dtype=dtype, device="cuda")
    tags0 = tags.clone()
    refs = np.zeros(P, np.int32)
    refs[ids] = 1
    table = np.full((2 * S, 1, 2), -1, np.int32)
    table[:S, 0, 0] = ids
    pages = ia.SequencePages(_i32(refs), _i32(table), _i32([5] * S + [0] * S), PS)
    if op == "grow":
        ia.fork_sequences(pages, _i32(range(S)), _i32(range(S, 2 * S)))
        ia.grow_sequences(pool, pages, _i32([0] * S + [1] * S), page_tags=tags, tag_map=tag_map, tag_default=3)
        at = slice(S, 2 * S)
        assert pages.table[:S, 0, 0].tolist() == ids.tolist() and int(pages.refs.max()) == 1
    else:
        assert int(ia.compact_pages(pool, pages, page_tags=tags, tag_map=tag_map, tag_default=3)) == S
        at = slice(0, S)
    new = pages.table[at, 0, 0].tolist()
    assert sorted(new) == list(range(S))
    want_tags = tags0.clone()
    for i, p in enumerate(new):
        want_tags[p] = tags0[int(ids[i])]
    assert torch.equal(tags, want_tags)
    for n, t in planes.items():
        want = before[n].clone()
        for i, p in enumerate(new):
            if n[2:] in PLANES[formats[i]]:
                want[p] = before[n][int(ids[i])]
        assert torch.equal(t.view(torch.uint8), want), n


@pytest.mark.parametrize("P", [(1 << 18) + 1, 300000, 800011])
def test_pools_of_several_runs_a_block(P):
    """More pages than a block of the plan holds in registers: free pages far apart, in every run, are found in order."""
    g = np.random.default_rng(P)
    PS, S, Ht, W = 1, 96, 8, 260
    pool, pages, want = _state(P, P, PS, S, Ht, W, g.integers(0, 200, S).tolist(), share=0.1, D=4)
    ia = _ia()
    # nearly all other pages in use by somebody else: the free ones are few and anywhere
    busy = (want.refs == 0) & (g.random(P) > 0.06)
    want.refs[busy] = 1
    pages.refs.copy_(_i32(want.refs))
    r = _counter()
    for _ in range(2):
        more = g.integers(0, 60, S)
        ia.grow_sequences(pool, pages, _i32(more), rejected=r)
        want.grow(more)
        _same(pool, pages, want)
        assert int(r) == want.rejected
    ia.free_sequences(pages, _i32(range(0, S, 3)))
    want.free(list(range(0, S, 3)))
    # (the others let go of theirs)
    want.refs[busy] = 0
    pages.refs[_i32(np.flatnonzero(busy)).long()] = 0
    assert int(ia.compact_pages(pool, pages)) == want.compact()
    _same(pool, pages, want)


def test_wants_beyond_31_bits():
    """Slots that together want more than 2^31 pages: those that the free pages reach grow, the sums do not wrap."""
    ia = _ia()
    S, W, P = 4096, 1 << 20, 3000
    table = torch.empty((S, 1, W), dtype=torch.int32, device="cuda")       # 17 GB; only entries of accepted slots are written
    pages = ia.SequencePages(torch.zeros(P, dtype=torch.int32, device="cuda"), table, _i32([0] * S), 1)
    pool = ia.PagePool(P, 1, 4, k_f16=torch.zeros(P, 1, 4, dtype=torch.float16, device="cuda"))
    more = np.full(S, W)
    more[:3] = [1000, 0, 1500]
    more[7] = -1
    r = _counter()
    ia.grow_sequences(pool, pages, _i32(more), rejected=r)
    assert pages.lengths.tolist() == [1000, 0, 1500] + [0] * (S - 3)
    assert int(r) == S - 3 and int(pages.refs.sum()) == 2500 and int(pages.refs[:2500].min()) == 1
    assert table[0, 0, :1000].tolist() == list(range(1000)) and table[2, 0, :1500].tolist() == list(range(1000, 2500))


def test_page_ops_captured():
    ia = _ia()
    pool, pages, want = _state(9, 4000, 16, 12, 4, 10, [100, 33, 64, 0, 0, 0, 0, 0, 0, 0, 0, 0], share=0.0)
    saved = [t.clone() for t in (pages.refs, pages.table, pages.lengths)]
    src, dst = _i32([0, 0, 1, 2]), _i32([5, 6, 7, 8])
    more, gone = _i32([1] * 12), _i32([0, 3])

    def step():
        ia.fork_sequences(pages, src, dst)
        ia.grow_sequences(pool, pages, more)
        ia.free_sequences(pages, gone)
        return ia.compact_pages(pool, pages)

    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        n = step()
    for t, s in zip((pages.refs, pages.table, pages.lengths), saved):
        t.copy_(s)
    for _ in range(2):                        # the second replay forks onto slots that hold tokens: refused
        gr.replay()
        want.fork([0, 0, 1, 2], [5, 6, 7, 8])
        want.grow([1] * 12)
        want.free([0, 3])
        assert int(n) == want.compact()
        _same(pool, pages, want)


def test_serving_run():
    """Prompt, decode, fork, copy-on-write, free and compact on one FP4 pool: every sequence keeps giving what
    attention over its own tokens gives."""
    ia = _ia()
    g = np.random.default_rng(4)
    P, PS, D, S, Ht, W, Hq = 600, 16, 128, 6, 2, 12, 8
    pool = ia.Fp4Pool.allocate(P, PS, D)
    pages = ia.SequencePages.allocate(P, PS, S, Ht, W)
    held = {s: (np.zeros((Ht, 0, D)), np.zeros((Ht, 0, D))) for s in range(S)}

    def write(counts):
        """New tokens of every slot: room, then rows."""
        n = max(counts)
        start = pages.lengths.clone()
        k = torch.randn(S, Ht, n, D, device="cuda", generator=gen).bfloat16()
        v = torch.randn(S, Ht, n, D, device="cuda", generator=gen).bfloat16()
        ia.grow_sequences(pool, pages, _i32(counts))
        ia.append_fp4(pool, k, v, pages.table, start, _i32(counts))
        for s in range(S):
            held[s] = tuple(np.concatenate([a, of.values(x[s, :, :counts[s]].double().cpu().numpy())], 1)
                            for a, x in zip(held[s], (k, v)))

    def check():
        q = torch.randn(S, Hq, D, device="cuda", generator=gen).half()
        got = ia.paged_decode_fp4(q, pool, pages.table, pages.lengths)
        for s in range(S):
            assert int(pages.lengths[s]) == held[s][0].shape[1]
            for h in range(Hq):
                k, v = (x[h // (Hq // Ht)] for x in held[s])
                want, A, reach = of.attention(q[s, h][None].double().cpu().numpy(), k, v,
                                              np.ones((1, k.shape[0]), bool), D ** -0.5)
                tol = A * (2.0 ** -11 + 2 * (D + 2) * 2.0 ** -24 * reach[:, None] + 2.0 ** -17) + 2.0 ** -11 * np.abs(want) + 2.0 ** -24
                assert (np.abs(got[s, h].double().cpu().numpy() - want) <= tol).all()

    gen = torch.Generator("cuda").manual_seed(1)
    write([37, 64, 100, 0, 0, 0])
    check()
    for _ in range(3):
        write([1, 1, 1, 0, 0, 0])
    check()
    write([4, 4, 4, 0, 0, 0])                     # draft tokens, most of them not kept
    ia.shrink_sequences(pages, _i32([3, 4, 1, 0, 0, 0]))
    for s, n in enumerate((3, 4, 1)):
        held[s] = tuple(x[:, :x.shape[1] - n] for x in held[s])
    check()
    ia.fork_sequences(pages, _i32([0, 0, 1]), _i32([3, 4, 5]))
    held[3], held[4], held[5] = held[0], held[0], held[1]
    check()
    write([1, 2, 0, 1, 3, 1])
    check()
    ia.free_sequences(pages, _i32([0, 2]))
    held[0] = held[2] = (np.zeros((Ht, 0, D)), np.zeros((Ht, 0, D)))
    n = ia.compact_pages(pool, pages)
    assert int(pages.table.max()) < int(n)
    check()
    write([50, 1, 0, 1, 1, 1])
    check()


def test_refused_growth_leaves_shared_pages_alone():
    """The documented step, with no page free for a copy: slot 2 shares slot 1's open page and was shrunk into it, so its
    new rows would be slot 1's tokens.  Slot 0 grows inside a page of its own."""
    ia = _ia()
    from intent_attention import sequence_pages
    PS, D, Ht, W = 16, 64, 2, 3
    P = 2 * Ht + Ht
    pool, pages = ia.Fp4Pool.allocate(P, PS, D), ia.SequencePages.allocate(P, PS, 3, Ht, W)
    gen = torch.Generator("cuda").manual_seed(3)

    def rows(n):
        return [torch.randn(3, Ht, n, D, device="cuda", generator=gen) for _ in range(2)]

    lines = sequence_pages.__doc__.split("loop::\n\n")[1].split("\n\n")[0]
    step = compile("\n".join(x.strip() for x in lines.splitlines()), "step", "exec")

    def run(n, new_tokens):
        k, v = rows(n)
        exec(step, dict(vars(ia), pool=pool, pages=pages, k_new=k, v_new=v, new_tokens=_i32(new_tokens)))
        return k, v

    k, v = run(20, [5, 20, 0])
    ia.fork_sequences(pages, _i32([1]), _i32([2]))
    ia.shrink_sequences(pages, _i32([0, 0, 2]))
    assert int((pages.refs == 0).sum()) == 0
    k2, v2 = run(1, [1, 0, 1])
    assert pages.lengths.tolist() == [6, 20, 18]
    for x, new, got in zip((k, v), (k2, v2), ia.read_fp4(pool, pages.table, None, 20, pages.lengths, dtype=torch.float32)):
        want = torch.zeros_like(got)
        held = torch.from_numpy(of.values(x.double().cpu().numpy())).float().cuda()
        want[0, :, :5], want[1], want[2, :, :18] = held[0, :, :5], held[1], held[1, :, :18]
        want[0, :, 5] = torch.from_numpy(of.values(new[0, :, 0].double().cpu().numpy())).float().cuda()
        assert torch.equal(got, want)


@pytest.mark.parametrize("view", ["heads_outside", "slices"])
def test_tables_with_strides(view):
    """The table as a view: heads outermost, or every other row of a wider one; what lies between stays."""
    ia = _ia()
    S, Ht, W = 7, 3, 6
    pool, pages, want = _state(11, 300, 16, S, Ht, W, [40, 17, 90, 0, 0, 5, 64], share=0.3)
    if view == "heads_outside":
        wide = pages.table.transpose(0, 1).contiguous()
        pages.table = wide.transpose(0, 1)
    else:
        wide = torch.full((2 * S, Ht + 1, W + 3), 77, dtype=torch.int32, device="cuda")
        wide[::2, 1:, 2:2 + W] = pages.table
        pages.table = wide[::2, 1:, 2:2 + W]
    r = _counter()
    more = [1, 15, 6, 3, 0, 40, 1]
    ia.grow_sequences(pool, pages, _i32(more), rejected=r)
    want.grow(more)
    ia.fork_sequences(pages, _i32([2]), _i32([4]), rejected=r)
    want.fork([2], [4])
    ia.shrink_sequences(pages, _i32([2, 0, 33, 1, 0, 0, 0]), rejected=r)
    want.shrink([2, 0, 33, 1, 0, 0, 0])
    ia.free_sequences(pages, _i32([0, 6]), rejected=r)
    want.free([0, 6])
    assert int(ia.compact_pages(pool, pages)) == want.compact()
    _same(pool, pages, want)
    assert int(r) == want.rejected
    if view == "slices":
        wide[::2, 1:, 2:2 + W] = 77
        assert (wide == 77).all()


def test_tables_that_overlap_are_refused():
    """An expanded table would give one entry to several slots or heads, each writing its own page into it."""
    ia = _ia()
    refs, ln = torch.zeros(8, dtype=torch.int32, device="cuda"), _i32([0, 0])
    one = torch.full((2, 1, 4), -1, dtype=torch.int32, device="cuda")
    for table in (one.expand(2, 3, 4), one[:1].expand(2, 1, 4), one.as_strided((2, 1, 4), (3, 4, 1)),
                  one.as_strided((2, 2, 2), (1, 2, 1)), one.as_strided((2, 2, 2), (2, 2, 1))):
        pages = ia.SequencePages(refs, table, ln, 16)
        pool = ia.Fp4Pool.allocate(8, 16, 64)
        for f in (lambda: ia.grow_sequences(pool, pages, ln), lambda: ia.free_sequences(pages, ln),
                  lambda: ia.compact_pages(pool, pages)):
            with pytest.raises(ValueError, match="overlap"):
                f()
    for table in (one.expand(2, 1, 4), one[:1], one[:, :, :1], one[:, :, :0], one[:0]):
        ia.SequencePages(refs, table, ln[:table.shape[0]], 16).struct()


def test_page_refusals():
    ia = _ia()
    pool, pages, _ = _state(1, 32, 16, 2, 1, 4, [10, 0])
    ok = _i32([1, 1])
    other = ia.SequencePages.allocate(31, 16, 2, 1, 4)
    bad = [
        lambda: ia.grow_sequences(pool, pages, _i32([1])),
        lambda: ia.shrink_sequences(pages, _i32([1])),
        lambda: ia.grow_sequences(pool, pages, ok.long()),
        lambda: ia.grow_sequences(pool, other, ok),
        lambda: ia.compact_pages(pool, ia.SequencePages.allocate(32, 8, 2, 1, 4)),
        lambda: ia.compact_pages(pool, pages, page_tags=torch.zeros(32, dtype=torch.uint8, device="cuda")),
        lambda: ia.compact_pages(pool, pages, page_tags=torch.zeros(3, dtype=torch.uint8, device="cuda"),
                                 tag_map=[0] * 16),
        lambda: ia.fork_sequences(pages, _i32([0, 1]), _i32([1])),
        lambda: ia.fork_sequences(pages, _i32([0]).long(), _i32([1])),
        lambda: ia.free_sequences(ia.SequencePages(pages.refs, pages.table[0], pages.lengths, 16), ok),
        lambda: ia.free_sequences(ia.SequencePages(pages.refs, pages.table, pages.lengths[:1], 16), ok),
        lambda: ia.free_sequences(pages, ok, rejected=torch.zeros(2, dtype=torch.int32, device="cuda")),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    with pytest.raises(RuntimeError):
        ia.fork_sequences(pages, torch.zeros(1, dtype=torch.int32), _i32([1]))
    ia.fork_sequences(pages, _i32([]), _i32([]))
    ia.free_sequences(pages, _i32([]))
