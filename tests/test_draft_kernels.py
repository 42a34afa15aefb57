"""The operators of drafted trees, each against its statement in 64 bits, and a step of all of them against decoding token
by token."""
import math
import random

import pytest
import torch

import kernel_references as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
NAN = float("nan")


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def status(dev):
    return torch.zeros(1, dtype=torch.int32, device=dev)


def ints(values, dev, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).to(dev)


def tree(rng, nodes, roots=1):
    """Parents and ancestors' bits of a random tree."""
    parents, bits = [], []
    for k in range(nodes):
        up = -1 if k < roots else rng.randrange(max(0, k - 6), k)
        parents.append(up)
        bits.append((bits[up] if up >= 0 else 0) | 1 << k)
    return parents, bits


def words_of(bits, count):
    return [(bits >> 64 * w & (1 << 64) - 1) - ((bits >> 64 * w + 63 & 1) << 64) for w in range(count)]


class Trees:
    """Trees of several requests over pages in no order; what no node may read is NaN."""

    def __init__(self, dev, heads, kv_heads, size, page, nodes, cached, dtype, seed, words=None, extra_rows=0, scale=1.0):
        rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
        self.nodes, self.cached, self.page, self.dev = nodes, cached, page, dev
        words = words or max(1, -(-max(nodes) // 64))
        bits, self.depth, self.parents = [], [], []
        for n in nodes:
            parents, b = tree(rng, n)
            bits += b
            self.parents += parents
            self.depth += [bin(x).count("1") - 1 for x in b]
        self.starts = [sum(nodes[:r]) for r in range(len(nodes) + 1)]
        rows = sum(nodes) + extra_rows
        self.mask = torch.zeros((rows, words), dtype=torch.int64)
        for i, b in enumerate(bits):
            self.mask[i] = torch.tensor(words_of(b, words))
        counts = [-(-(c + n) // page) for c, n in zip(cached, nodes)]
        order = torch.randperm(sum(counts) + 3, generator=gen).tolist()
        width = max(counts + [1]) + 1
        table, at = torch.full((len(nodes), width), -1, dtype=torch.int32), 0
        for r, c in enumerate(counts):
            table[r, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
            at += c
        pages = sum(counts) + 3
        self.k = torch.full((pages, kv_heads, page, size), NAN)
        self.v = torch.full((pages, kv_heads, page, size), NAN)
        for r, (c, n) in enumerate(zip(cached, nodes)):
            for j in range(c + n):
                self.k[table[r, j // page], :, j % page] = torch.randn((kv_heads, size), generator=gen)
                self.v[table[r, j // page], :, j % page] = torch.randn((kv_heads, size), generator=gen)
        self.q = (torch.randn((rows, heads, size), generator=gen) * scale).to(dtype)
        self.k, self.v, self.table = self.k.to(dtype), self.v.to(dtype), table
        first = [c for c, n in zip(cached, nodes) for _ in range(n)]
        self.positions = [c + d for c, d in zip(first, self.depth)] + [0] * extra_rows
        self.scale = size ** -0.5

    def slot(self, request, place):
        return int(self.table[request, place // self.page]), place % self.page

    def arguments(self):
        d = self.dev
        return (self.q.to(d), self.k.to(d), self.v.to(d), self.table.to(d), ints(self.starts, d), ints(self.cached, d), self.mask.to(d))

    def run(self, **options):
        from einf_b200 import ops

        q, *rest = self.arguments()
        out, st = torch.full_like(q, 7.0), status(self.dev)
        if "window" in options:
            options["positions"] = ints(self.positions, self.dev)
        ops.tree_attention(q, *rest, out, self.scale, st, **options)
        assert int(st) == 0
        return out

    def check(self, got, window=None, softcap=None):
        want, bound = ref.tree_attention(self.q, self.k, self.v, self.table, torch.tensor(self.starts), torch.tensor(self.cached),
                                         self.mask, self.scale, self.positions, window, softcap)
        got = got.double().cpu()
        live = self.starts[-1]
        assert torch.equal(got[live:], torch.full_like(got[live:], 7.0)), "rows of no request were written"
        got, want, bound = got[:live], want[:live], bound[:live]
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[got.isinf()])
        fine = want.isfinite()
        if self.q.dtype == torch.bfloat16:
            # the weights as the second product's operand and the result are rounded once each, by half a step of 2^-7
            bound = bound + self.weights_step(window, softcap) + want.abs() * 2.0 ** -8
        off = ((got - want).abs() - bound * 1.0001)[fine]
        assert off.numel() == 0 or float(off.max()) <= 0, f"off by {float(off.max())} more than may be"

    def weights_step(self, window, softcap):
        """2^-8 of the sum of the values' sizes, weighted."""
        sizes, _ = ref.tree_attention(self.q, self.k, self.v.abs(), self.table, torch.tensor(self.starts), torch.tensor(self.cached),
                                      self.mask, self.scale, self.positions, window, softcap)
        return sizes[:self.starts[-1]] * 2.0 ** -8 * 1.01


LAYOUTS = [
    # heads, kv heads, head size, page, nodes, cached
    (4, 2, 48, 4, [5, 1, 7], [13, 0, 40]),
    (14, 2, 64, 16, [8], [129]),
    (14, 2, 64, 16, [1, 19, 3, 0, 40], [0, 1, 127, 9, 300]),
    (12, 2, 128, 16, [16, 5], [260, 31]),
    (28, 4, 128, 32, [37], [128]),
    (6, 6, 64, 8, [3, 65], [70, 5]),
    (3, 1, 20, 5, [2, 9], [33, 64]),
    (40, 1, 33, 7, [4], [50]),
    (2, 1, 256, 16, [6, 2], [100, 3]),
    (1, 1, 1, 1, [3], [2]),
    (8, 1, 128, 64, [33, 70], [63, 1]),
    (130, 1, 64, 16, [3], [40]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads, size, page, nodes, cached", LAYOUTS)
def test_tree_attention(dev, dtype, heads, kv_heads, size, page, nodes, cached):
    case = Trees(dev, heads, kv_heads, size, page, nodes, cached, dtype, seed=heads + size, extra_rows=2)
    case.check(case.run())
    case.check(case.run(max_nodes=max(nodes), max_cached=max(cached)))
    # what the caller says of the sizes is no more than a hint
    case.check(case.run(max_nodes=1, max_cached=0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads, size, page, nodes, cached", [LAYOUTS[0], LAYOUTS[2], LAYOUTS[3], LAYOUTS[6]])
@pytest.mark.parametrize("window, softcap", [(1, None), (2, 3.0), (30, None), (200, 20.0), (10 ** 9, None)])
def test_tree_attention_with_a_window_and_a_cap(dev, dtype, heads, kv_heads, size, page, nodes, cached, window, softcap):
    case = Trees(dev, heads, kv_heads, size, page, nodes, cached, dtype, seed=3)
    for r, c in enumerate(cached):      # pages that the windows have passed are given back
        for gone in range(max(0, c - window + 1) // page):
            case.table[r, gone] = -1
    given = case.table.clone()
    got = case.run(window=window, **({"softcap": softcap} if softcap else {}))
    case.table = given.clamp(min=0)     # the statement looks them up before it leaves them out
    case.check(got, window, softcap)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads, size, page", [(4, 2, 48, 4), (14, 2, 64, 16), (12, 2, 128, 16)])
def test_masks_that_are_no_tree(dev, dtype, heads, kv_heads, size, page):
    """Rows that see nothing, a row that sees all nodes, bits of nodes that a request does not have."""
    case = Trees(dev, heads, kv_heads, size, page, [9, 4, 3], [0, 17, 0], dtype, seed=8, words=2)
    case.mask[2] = 0
    case.mask[5, 0], case.mask[5, 1] = -1, -1
    case.mask[9] = 0
    case.mask[11, 0] = -1
    case.mask[13:] = 0
    got = case.run()
    assert torch.equal(got[2], torch.zeros_like(got[2])) and torch.equal(got[13:], torch.zeros_like(got[13:]))
    case.check(got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads, size, page", [(4, 2, 48, 4), (14, 2, 64, 16), (12, 2, 128, 16)])
@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(dev, dtype, heads, kv_heads, size, page, bad):
    case = Trees(dev, heads, kv_heads, size, page, [12, 6], [150, 40], dtype, seed=11)
    sibling = next(k for k in range(1, 12) if any(not int(case.mask[j, 0]) >> k & 1 for j in range(k + 1, 12)))
    page_of, row = case.slot(0, 150 + sibling)
    case.v[page_of, 0, row, ::3] = bad
    page_of, row = case.slot(1, 40 + 3)
    case.k[page_of, kv_heads - 1, row, 1] = bad
    got = case.run().double().cpu()
    clean = Trees(dev, heads, kv_heads, size, page, [12, 6], [150, 40], dtype, seed=11)
    want = clean.run().double().cpu()
    group = heads // kv_heads
    for j in range(12):
        sees = int(case.mask[j, 0]) >> sibling & 1
        mine = got[j, :group]
        if sees:
            assert not mine[:, ::3].isfinite().any() and torch.equal(mine[:, 1::3], want[j, :group, 1::3])
        else:
            assert torch.equal(mine, want[j, :group])
        assert torch.equal(got[j, group:], want[j, group:])
    for j in range(12, 18):
        if int(case.mask[j, 0]) >> 3 & 1:
            last = got[j, heads - group:]
            if math.isnan(bad):
                assert last.isnan().all()
        else:
            assert torch.equal(got[j], want[j])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads, size, page", [(4, 2, 48, 4), (14, 2, 64, 16), (12, 2, 128, 16)])
def test_scores_far_apart(dev, dtype, heads, kv_heads, size, page):
    """Scores of several hundred: late keys that outweigh all before them, rows whose first tile is far below the rest."""
    case = Trees(dev, heads, kv_heads, size, page, [7, 20], [333, 200], dtype, seed=5, scale=25.0)
    case.check(case.run())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads, size, page", [(4, 2, 48, 4), (14, 2, 64, 16), (12, 2, 128, 16)])
@pytest.mark.parametrize("nodes, cached", [([5], [700]), ([30, 3], [390, 1100])])
def test_scores_that_rise_and_fall_along_the_keys(dev, dtype, heads, kv_heads, size, page, nodes, cached):
    """One direction for all queries and keys, so that the scores are what is asked for: hundreds above those of the first keys
    later on; hundreds below zero for all of them; the first tiles outside the window and the rest far below zero; one key at 9,000."""
    def run(levels, **options):
        case = Trees(dev, heads, kv_heads, size, page, nodes, cached, dtype, seed=6)
        case.q[:] = 1.0
        for r, (c, n) in enumerate(zip(cached, nodes)):
            for j in range(c + n):
                where, row = case.slot(r, j)
                case.k[where, :, row] = torch.tensor(levels(j, c)).to(dtype).float().item() * size ** -0.5
        case.check(case.run(**options), options.get("window"))

    run(lambda j, c: -100.0 if j < 200 else 150.0 + j % 3)
    run(lambda j, c: 150.0 if j < 200 else -100.0)
    run(lambda j, c: -300.0 - j % 5)
    run(lambda j, c: 40.0 if j < 300 else -250.0, window=200)
    run(lambda j, c: 9000.0 if j == 350 else 8999.0 if j == 30 else 0.5 * (j % 7))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [48, 128])
def test_a_result_does_not_depend_on_the_call(dev, dtype, size):
    """The same call twice gives the same bits, on another stream and from a captured graph too."""
    from einf_b200 import ops

    case = Trees(dev, 12, 2, size, 16, [9, 30, 2], [500, 77, 1200], dtype, seed=2)
    first = case.run()
    assert torch.equal(first, case.run())
    arguments, st = case.arguments(), status(dev)
    outs = [torch.zeros_like(first) for _ in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.tree_attention(*arguments, outs[0], case.scale, st)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for out in outs[1:]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.tree_attention(*arguments, out, case.scale, st)
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for graph, stream in zip(graphs, streams):      # both at once
        with torch.cuda.stream(stream):
            for _ in range(5):
                graph.replay()
    torch.cuda.synchronize()
    assert int(st) == 0 and all(torch.equal(first, out) for out in outs)


FAR = (1 << 31) + 5      # elements: offsets beyond 32 bits behind them


@pytest.mark.parametrize("heads, kv_heads, size, page", [(12, 2, 128, 16), (4, 2, 48, 5)])
def test_pages_beyond_32_bits(dev, heads, kv_heads, size, page):
    """The pages at the end of a cache of more than 2^31 elements give the bits that they give in a small one."""
    from einf_b200 import ops

    case = Trees(dev, heads, kv_heads, size, page, [9, 30], [77, 400], torch.bfloat16, seed=3)
    want = case.run()
    q, k, v, table, *rest = case.arguments()
    before = FAR // (kv_heads * page * size) + 1
    far = [torch.empty((before + t.shape[0],) + tuple(t.shape[1:]), dtype=t.dtype, device=dev) for t in (k, v)]
    for big, t in zip(far, (k, v)):
        big[before:] = t
    out, st = torch.full_like(q, 7.0), status(dev)
    ops.tree_attention(q, *far, torch.where(table < 0, table, table + before), *rest, out, case.scale, st)
    assert int(st) == 0 and torch.equal(out, want)
    small, kept, path = [k, v], ints([5, 3], dev), ints([[0, 2, 3, 6, 8], [0, 1, 29, -1, -1]], dev)
    ops.move_accepted(ops.CacheRows(small), table, rest[1], path, kept, st)
    ops.move_accepted(ops.CacheRows(far), torch.where(table < 0, table, table + before), rest[1], path, kept, st)
    assert int(st) == 0
    for big, t in zip(far, small):
        assert torch.equal(big[before:].view(torch.int16), t.view(torch.int16))


@pytest.mark.parametrize("vocab", [151936, 151935])
def test_logits_beyond_32_bits(dev, vocab):
    case = logits_case(dev, vocab, [2, 3], 50, seed=1, biases=4, nodes=True)
    want = shape(dev, case)
    before = FAR // vocab + 1
    big = torch.empty((before + 5, vocab), device=dev)
    big[before:] = case.pop("logits").to(dev)
    on, st = {name: t.to(dev) for name, t in case.items()}, status(dev)
    starts = on.pop("row_start") + before
    for name in ("tree_mask", "node_tokens"):
        t = on[name]
        on[name] = torch.zeros((before + 5,) + tuple(t.shape[1:]), dtype=t.dtype, device=dev)
        on[name][before:] = t
    from einf_b200 import ops

    ops.shape_logits(big, big, starts, st, **on)
    assert int(st) == 0 and torch.equal(big[before:], want)


@pytest.mark.parametrize("dtype, size", [(torch.float32, 20), (torch.bfloat16, 64)])
def test_a_window_wider_than_any_context_is_none(dev, dtype, size):
    from einf_b200 import ops

    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(s, generator=gen).to(dtype).to(dev) for s in ((5, 4, size), (40, 2, 8, size), (40, 2, 8, size)))
    mask = torch.tensor([[1], [3], [5], [11], [1]], dtype=torch.int64, device=dev)
    outs = []
    for window in (None, 1 << 40, (1 << 31) - 1):
        out, st = torch.full_like(q, 3.0), status(dev)
        ops.tree_attention(q, k, v, ints([list(range(40)), list(range(40))], dev), ints([0, 4, 5], dev), ints([300, 0], dev), mask, out, 0.2, st,
                           positions=ints([300, 301, 301, 302, 0], dev), window=window)
        assert int(st) == 0
        outs.append(out.cpu())
    assert outs[0].isfinite().all()
    # the same keys, weighed in other orders: sums of up to 304 products in 32 bits, probabilities of bfloat16 rounded
    # against other references (2^-8 each), outputs rounded once more (2^-8)
    bound = 304 * 2.0 ** -24 if dtype == torch.float32 else 3 * 2.0 ** -8
    top = float(v.float().abs().max())
    for out in outs[1:]:
        assert ((out.double() - outs[0].double()).abs() <= bound * top).all()


def test_bad_pages_and_lengths_set_the_status_word(dev):
    from einf_b200 import ops

    for dtype, size in ((torch.float32, 48), (torch.bfloat16, 48), (torch.bfloat16, 64), (torch.bfloat16, 128)):
        for fault in ("page", "negative page", "cached", "negative cached"):
            case = Trees(dev, 4, 2, size, 16, [5, 3], [50, 20], dtype, seed=1)
            if fault == "page":
                case.table[1, 1] = 10 ** 6
            elif fault == "negative page":
                case.table[1, 0] = -1
            else:
                case.cached[1] = 10 ** 9 if fault == "cached" else -5
            arguments, st = case.arguments(), status(dev)
            out = torch.zeros_like(arguments[0])
            ops.tree_attention(*arguments, out, case.scale, st)
            assert int(st) == ops.STATUS_BAD_PAGE
            case.cached = [50, 20]
            want, _ = ref.tree_attention(case.q[:5], case.k, case.v, case.table[:1], torch.tensor([0, 5]), torch.tensor([50]),
                                         case.mask[:5], case.scale)
            torch.testing.assert_close(out[:5].double().cpu(), want, rtol=2e-2, atol=2e-2)     # the other request is not touched by it


# ---------------------------------------------------------------------------
def logits_case(dev, vocab, rows_of, capacity, seed, biases=0, nodes=False, masks=None, history=True):
    gen, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    rows, requests = sum(rows_of), len(rows_of)
    case = dict(logits=torch.randn((rows, vocab), generator=gen) * 5,
                row_start=torch.tensor([sum(rows_of[:r]) for r in range(requests + 1)], dtype=torch.int32))
    if history:
        case["history"] = torch.randint(0, max(1, vocab // 3), (requests, capacity), generator=gen, dtype=torch.int32)
        case["history_lens"] = torch.tensor([rng.randint(0, capacity) for _ in rows_of], dtype=torch.int32)
        case["prompt_lens"] = torch.tensor([rng.randint(0, int(n)) for n in case["history_lens"]], dtype=torch.int32)
        # what stands behind a history's end is no token
        for r, n in enumerate(case["history_lens"].tolist()):
            case["history"][r, n:] = -77
    case["repetition"] = torch.rand(requests, generator=gen) + 0.6
    case["presence"] = torch.randn(requests, generator=gen)
    case["frequency"] = torch.randn(requests, generator=gen)
    if nodes:
        bits = [b for n in rows_of for b in tree(rng, n)[1]]
        words = max(1, -(-max(rows_of) // 64))
        case["tree_mask"] = torch.tensor([words_of(b, words) for b in bits] or [[0] * words], dtype=torch.int64).view(-1, words)
        case["node_tokens"] = torch.randint(0, min(vocab, 9), (rows,), generator=gen, dtype=torch.int32) * (vocab // min(vocab, 9))
    if biases:
        case["bias_ids"] = torch.randint(-1, vocab, (requests, biases), generator=gen, dtype=torch.int32)
        case["bias"] = torch.randn((requests, biases), generator=gen) * 3
    if masks is not None:
        count = rows if masks == "rows" else 2
        case["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (count, -(-vocab // 32)), generator=gen).to(torch.int32)
        if masks == "shared":
            case["allowed_rows"] = torch.tensor([rng.choice([-1, 0, 1]) for _ in range(rows)], dtype=torch.int32)
    return case


def shape(dev, case, out=None):
    from einf_b200 import ops

    on = {name: t.to(dev) for name, t in case.items()}
    logits, starts, st = on.pop("logits"), on.pop("row_start", None), status(dev)
    out = logits if out == "in place" else torch.full_like(logits, 7.0)
    ops.shape_logits(logits, out, starts, st, **on)
    assert int(st) == 0
    return out


def check_logits(case, got, untouched=7.0):
    """Five rounded operations on values of at most `size`, each off by 2^-24 of what it gives."""
    want = ref.shape_logits(case["logits"], case.get("row_start"), **{n: t for n, t in case.items() if n not in ("logits", "row_start")})
    got = got.double().cpu()
    nobody = want.isnan() & ~case["logits"].isnan()
    before = torch.full_like(got, untouched) if untouched is not None else case["logits"].double()
    assert torch.equal(got[nobody], before[nobody])
    got, want = got[~nobody], want[~nobody]
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    # a factor of less than two; then what may be taken off and added
    sizes = case["logits"].double()[~nobody].abs() * 2
    extra = sum(float(case[name].abs().max()) for name in ("presence", "bias") if name in case)
    if "frequency" in case:
        answered = (case["history"].shape[1] if "history" in case else 0) + (case["logits"].shape[0] if "node_tokens" in case else 0)
        extra += float(case["frequency"].abs().max()) * answered
    assert ((got - want).abs() <= 5 * 2.0 ** -24 * (sizes + extra))[fine].all()


@pytest.mark.parametrize("vocab, rows_of, capacity", [
    (50, [1, 1, 1], 40), (331, [3, 0, 9], 100), (3001, [1], 1), (2003, [70], 500), (4100, [2, 5], 333), (40000, [1, 2], 64), (1, [2], 5),
    (32, [1, 1], 8),
])
@pytest.mark.parametrize("biases, nodes, masks", [(0, False, None), (7, True, "rows"), (0, True, None), (3, False, "shared"), (1, True, "shared")])
def test_shape_logits(dev, vocab, rows_of, capacity, biases, nodes, masks):
    case = logits_case(dev, vocab, rows_of, capacity, seed=vocab + biases, biases=biases, nodes=nodes, masks=masks)
    want = shape(dev, case)
    check_logits(case, want)
    assert torch.equal(shape(dev, case, "in place"), want)


@pytest.mark.parametrize("vocab", [2003, 2100])
def test_shape_logits_of_many_nodes_with_few_tokens(dev, vocab):
    """All hits of a token in one CTA, every node on some row's path."""
    case = logits_case(dev, vocab, [700, 2], 20, seed=5, nodes=True, masks="shared")
    case["node_tokens"] = case["node_tokens"] % 5
    case["tree_mask"][::3] = -1
    check_logits(case, shape(dev, case))


def test_shape_logits_with_one_thing_alone(dev):
    full = logits_case(dev, 700, [1, 1, 1], 30, seed=4, biases=5, masks="rows")
    del full["row_start"]      # a row each
    for names in (["allowed"], ["bias_ids", "bias"], ["history", "history_lens", "repetition"], ["history", "history_lens", "prompt_lens", "presence"],
                  ["history", "history_lens", "frequency"], ["history", "history_lens"], []):
        case = {n: full[n] for n in ["logits"] + names}
        check_logits(case, shape(dev, case))


def test_rows_of_no_request_keep_what_they_hold(dev):
    case = logits_case(dev, 333, [2, 3], 20, seed=9, nodes=True, masks="rows", biases=2)
    for name in ("logits", "tree_mask", "node_tokens", "allowed"):
        pad = torch.ones_like(case[name][:1])
        case[name] = torch.cat([pad, case[name], pad, pad])
    case["row_start"] += 1
    check_logits(case, shape(dev, case))


def test_logits_that_are_not_finite(dev):
    case = logits_case(dev, 97, [2, 2], 60, seed=6, nodes=True, masks="rows", biases=4)
    lowest = torch.finfo(torch.float32).min
    case["logits"][0, ::7], case["logits"][1, ::5], case["logits"][2, ::3], case["logits"][3, ::4] = NAN, math.inf, -math.inf, lowest
    case["repetition"] = torch.tensor([1.0, 0.5])       # twice the lowest value would not be finite
    case["logits"][3] = case["logits"][3].clamp(min=lowest / 4)
    case["bias"][1, 0] = -math.inf
    case["allowed"][1] = 0                              # nothing may come
    got = shape(dev, case)
    assert (got[1] == -math.inf).all()
    want = ref.shape_logits(case["logits"], case["row_start"], **{n: t for n, t in case.items() if n not in ("logits", "row_start")})
    torch.testing.assert_close(got.double().cpu(), want, rtol=1e-6, atol=1e-4, equal_nan=True)


def test_bad_tokens_and_masks_set_the_status_word(dev):
    from einf_b200 import ops

    for name, value, word in (("history", 97, "BAD_TOKEN"), ("history", -1, "BAD_TOKEN"), ("node_tokens", 97, "BAD_TOKEN"), ("bias_ids", 1 << 30, "BAD_TOKEN"),
                              ("allowed_rows", 2, "BAD_INDEX")):
        case = logits_case(dev, 97, [2, 2], 60, seed=6, nodes=True, masks="shared", biases=4)
        case["history_lens"][:] = 60
        case["history"].clamp_(min=0)
        clean = shape(dev, {n: t.clone() for n, t in case.items()})
        case[name].view(-1)[-1] = value
        on = {n: t.to(dev) for n, t in case.items()}
        st, out = status(dev), torch.zeros((4, 97), device=dev)
        ops.shape_logits(on.pop("logits"), out, on.pop("row_start"), st, **on)
        assert int(st) == getattr(ops, f"STATUS_{word}")
        assert torch.equal(out[:2], clean[:2])


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("nodes", [[1], [0, 5, 0], [64, 1, 33], [200, 3], [1024, 1025, 1500], [7] * 300])
@pytest.mark.parametrize("depth", [1, 3, 40])
def test_accept_drafts(dev, nodes, depth):
    from einf_b200 import ops

    rng = random.Random(sum(nodes) + depth)
    parents, tokens, targets = [], [], []
    for n in nodes:
        up, _ = tree(rng, n)
        words = [rng.randrange(4) for _ in range(n)]
        want = [rng.randrange(4) for _ in range(n)]
        for k in range(1, n):
            if rng.random() < 0.8:
                want[up[k]] = words[k]
            if rng.random() < 0.05:      # no node's child
                up[k] = rng.choice([-1, k, k + 1, n + 7, -9])
        parents += up
        tokens += words
        targets += want
    starts = [sum(nodes[:r]) for r in range(len(nodes) + 1)]
    given = [ints(v, dev) for v in (tokens, targets, parents, starts)]
    path, answer = torch.full((len(nodes), depth), 9, dtype=torch.int32, device=dev), torch.full((len(nodes), depth), 9, dtype=torch.int32, device=dev)
    counts = torch.full((len(nodes),), 9, dtype=torch.int32, device=dev)
    ops.accept_drafts(*given, path, answer, counts)
    want = ref.accept_drafts(*(t.cpu() for t in given), depth)
    assert (path.tolist(), answer.tolist(), counts.tolist()) == want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shapes, page", [([(2, 64)] * 6, 16), ([(1, 3), (2, 20), (3, 8)], 5), ([(2, 16)] * 200, 4), ([(1, 1)], 1)])
def test_move_accepted(dev, dtype, shapes, page):
    """Paths whose places lie on other kept nodes' places, paths that move nothing, over page borders."""
    from einf_b200 import ops

    rng, gen = random.Random(page), torch.Generator().manual_seed(page)
    nodes, cached = [20, 1, 90, 6, 2], [7, 0, 33, 15, 64]
    counts = [-(-(c + n) // page) for c, n in zip(cached, nodes)]
    order, table, at = torch.randperm(sum(counts), generator=gen).tolist(), [], 0
    for c in counts:
        table.append(order[at:at + c] + [-1] * (max(counts) - c))
        at += c
    paths = [[0, 2, 3, 4, 19], [0], [0] + sorted(rng.sample(range(1, 90), 75)), [0, 1, 2, 3, 4, 5], [0, 1]]
    depth = 80
    path = torch.tensor([p + [-1] * (depth - len(p)) for p in paths], dtype=torch.int32)
    kept = torch.tensor([len(p) for p in paths], dtype=torch.int32)
    caches = [torch.randn((sum(counts), heads, page, size), generator=gen).to(dtype) for heads, size in shapes]
    want = ref.move_accepted(caches, torch.tensor(table), torch.tensor(cached), path, kept)
    on, st = [c.to(dev) for c in caches], status(dev)
    ops.move_accepted(ops.CacheRows(on), ints(table, dev), ints(cached, dev), path.to(dev), kept.to(dev), st)
    assert int(st) == 0
    assert all(torch.equal(a.cpu(), b) for a, b in zip(on, want))


def test_move_accepted_leaves_what_it_cannot_place(dev):
    from einf_b200 import ops

    for path, table, word in (([0, 4, 3, 5], [0, 1], "BAD_INDEX"), ([0, 4, 4], [0, 1], "BAD_INDEX"), ([0, -1, 6], [0, 1], "BAD_INDEX"),
                              ([0, 3, 40], [0, 1], "BAD_PAGE"), ([0, 3, 6], [0, 5], "BAD_PAGE"), ([0, 3, 6], [0, -1], "BAD_PAGE")):
        cache = torch.arange(2 * 8 * 4, dtype=torch.float32).view(2, 1, 8, 4).to(dev)
        before, st = cache.clone(), status(dev)
        ops.move_accepted(ops.CacheRows([cache]), ints([table], dev), ints([4], dev), ints([path], dev), ints([len(path)], dev), st)
        assert int(st) == getattr(ops, f"STATUS_{word}")
        assert torch.equal(cache[0, 0, :5], before[0, 0, :5])


# ---------------------------------------------------------------------------
class Decoder:
    """Two layers of attention with a residual between an embedding and itself as the output matrix: enough of a model that
    a wrong key, position, mask or count shows in its tokens."""

    def __init__(self, vocab=97, heads=4, kv_heads=2, size=16, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.vocab, self.heads, self.kv_heads, self.size, width = vocab, heads, kv_heads, size, 48
        self.embedding = torch.randn((vocab, width), generator=gen)
        self.qkv = [torch.randn((width, (heads + 2 * kv_heads) * size), generator=gen) * 0.3 for _ in range(2)]
        self.output = [torch.randn((heads * size, width), generator=gen) * 0.5 for _ in range(2)]
        self.inv_freq = 100.0 ** (-torch.arange(0, size, 2).float() / size)

    def rotate(self, x, positions):
        angle = positions[:, None, None].double() * self.inv_freq.double()
        a, b = x.chunk(2, -1)
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)

    def logits(self, tokens):
        """Of the last of a sequence's tokens, all of them recomputed, in 64 bits."""
        h, positions = self.embedding.double()[tokens], torch.arange(len(tokens))
        for qkv, output in zip(self.qkv, self.output):
            x = (h @ qkv.double()).view(len(tokens), -1, self.size)
            q, k = self.rotate(x[:, :self.heads], positions), self.rotate(x[:, self.heads:self.heads + self.kv_heads], positions)
            k, v = (t.repeat_interleave(self.heads // self.kv_heads, 1) for t in (k, x[:, self.heads + self.kv_heads:]))
            s = torch.einsum("ihd,jhd->hij", q, k) * self.size ** -0.5
            s = s.masked_fill(torch.ones(len(tokens), len(tokens)).triu(1).bool(), -math.inf)
            h = h + torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).reshape(len(tokens), -1) @ output.double()
        return h[-1] @ self.embedding.double().T


def test_drafted_steps_answer_what_decoding_token_by_token_answers(dev):
    """Three requests with penalties, biases and masks: every step drafts a tree (with the right tokens on one branch as far as
    luck has it), verifies it, keeps the agreed path and closes the gaps in the cache; what it answers is what the plain
    model, one token at a time, answers."""
    from einf_b200 import ops

    model, rng, page, steps = Decoder(), random.Random(5), 4, 8
    prompts = [[3, 14, 15, 92, 6], [53], [58, 9, 79, 32, 38, 46, 26]]
    requests, capacity, heads, kv_heads, size = 3, 96, model.heads, model.kv_heads, model.size
    penalties = dict(repetition=torch.tensor([1.3, 1.0, 1.1]), presence=torch.tensor([0.5, 0.0, 0.7]), frequency=torch.tensor([0.1, 0.3, 0.0]))
    bias_ids, bias = torch.tensor([[5, -1], [60, 61], [-1, 8]], dtype=torch.int32), torch.tensor([[9.0, 0.0], [4.0, -3.0], [0.0, 6.0]])
    allowed = torch.randint(-2 ** 31, 2 ** 31, (2, 4), generator=torch.Generator().manual_seed(3)).to(torch.int32)
    mask_of = [0, -1, 1]

    def next_plain(r, tokens):
        case = dict(logits=model.logits(tokens)[None], history=torch.tensor([tokens]), history_lens=torch.tensor([len(tokens)]),
                    prompt_lens=torch.tensor([len(prompts[r])]), bias_ids=bias_ids[r:r + 1], bias=bias[r:r + 1], allowed=allowed,
                    allowed_rows=torch.tensor([mask_of[r]]), **{n: t[r:r + 1] for n, t in penalties.items()})
        return int(ref.shape_logits(row_start=None, **case)[0].argmax())

    plain = []
    for r, prompt in enumerate(prompts):
        tokens = list(prompt)
        for _ in range(capacity - 30):
            tokens.append(next_plain(r, tokens))
        plain.append(tokens)
    pages = requests * capacity // page
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).view(requests, -1).int()
    caches = [(torch.full((pages, kv_heads, page, size), NAN, device=dev), torch.full((pages, kv_heads, page, size), NAN, device=dev)) for _ in range(2)]
    rows_of_cache = ops.CacheRows([t for pair in caches for t in pair])
    on = {n: t.to(dev) for n, t in dict(penalties, bias_ids=bias_ids, bias=bias, allowed=allowed, table=table).items()}
    embedding, st = model.embedding.to(dev), status(dev)
    history = torch.zeros((requests, capacity), dtype=torch.int32)
    sequences, cached = [list(p) for p in prompts], [0, 0, 0]
    kept_total = 0
    for step in range(steps):
        tokens, parents, bits, nodes = [], [], [], []
        for r in range(requests):
            if step == 0:       # the prompt: a tree without branches
                line, up = list(prompts[r]), list(range(-1, len(prompts[r]) - 1))
            else:
                line, up = [sequences[r][-1]], [-1]
                done, depth, node = len(sequences[r]), 0, 0
                for k in range(1, rng.randint(2, 12)):
                    if rng.random() < 0.6 and done + depth < len(plain[r]):       # the right branch goes on
                        line.append(plain[r][done + depth])
                        up.append(node)
                        node, depth = k, depth + 1
                    else:
                        line.append(rng.randrange(model.vocab))
                        up.append(rng.randrange(k))
            chain = []
            for k, parent in enumerate(up):
                chain.append((chain[parent] if parent >= 0 else 0) | 1 << k)
            tokens += line
            parents += up
            bits += chain
            nodes.append(len(line))
        starts = [sum(nodes[:r]) for r in range(requests + 1)]
        first = [c for c, n in zip(cached, nodes) for _ in range(n)]
        positions = [c + bin(b).count("1") - 1 for c, b in zip(first, bits)]
        slots = []
        for r in range(requests):
            slots += [int(table[r, (cached[r] + k) // page]) * page + (cached[r] + k) % page for k in range(nodes[r])]
        node_tokens, q_start, lens = ints(tokens, dev), ints(starts, dev), ints(cached, dev)
        tree_mask, place, where = ints([[b] for b in bits], dev, torch.int64), ints(positions, dev), ints(slots, dev)
        h = embedding[node_tokens.long()]
        for layer, (k_cache, v_cache) in enumerate(caches):
            q = torch.empty((len(tokens), heads, size), device=dev)
            ops.rope_kv_write(h @ model.qkv[layer].to(dev), None, place, model.inv_freq.to(dev), where, q, k_cache, v_cache, heads, kv_heads, size, st)
            mixed = torch.empty_like(q)
            ops.tree_attention(q, k_cache, v_cache, on["table"], q_start, lens, tree_mask, mixed, size ** -0.5, st)
            h = h + mixed.flatten(1) @ model.output[layer].to(dev)
        logits = h @ embedding.T
        # a node's path counts on its own: the history ends before the root, whose token is the tree's
        for r in range(requests):
            history[r, :cached[r]] = torch.tensor(sequences[r][:cached[r]], dtype=torch.int32)
        prompt_rows = step == 0
        ops.shape_logits(
            logits, logits, q_start, st, history=history.to(dev), history_lens=lens,
            prompt_lens=ints([min(len(p), c) for p, c in zip(prompts, cached)], dev),
            node_tokens=None if prompt_rows else node_tokens, tree_mask=None if prompt_rows else tree_mask, bias_ids=on["bias_ids"], bias=on["bias"],
            allowed=on["allowed"], allowed_rows=ints([mask_of[r] for r in range(requests) for _ in range(nodes[r])], dev),
            **{n: on[n] for n in penalties})
        if prompt_rows:       # the prompt's tokens are no drafts: its last row alone is asked, with the prompt as history
            shaped = []
            for r, prompt in enumerate(prompts):
                shaped.append(next_plain(r, prompt))
                assert shaped[r] == plain[r][len(prompt)]
                sequences[r].append(shaped[r])
                cached[r] = len(prompt)
            continue
        targets = torch.empty(len(tokens), dtype=torch.int32, device=dev)
        ops.argmax(logits, targets)
        path, answer = (torch.empty((requests, 12), dtype=torch.int32, device=dev) for _ in range(2))
        counts = torch.empty(requests, dtype=torch.int32, device=dev)
        ops.accept_drafts(node_tokens, targets, ints(parents, dev), q_start, path, answer, counts)
        ops.move_accepted(rows_of_cache, on["table"], lens, path, counts, st)
        assert int(st) == 0
        for r, n in enumerate(counts.tolist()):
            sequences[r] += answer[r, :n].tolist()
            assert answer[r, n:].tolist() == [-1] * (12 - n)
            assert sequences[r] == plain[r][:len(sequences[r])], f"step {step}, request {r}"
            cached[r] += n
            kept_total += n
    assert kept_total > 2 * requests * (steps - 1)      # drafts were kept


@pytest.mark.parametrize("size", [64, 128])
def test_a_decode_step_behind_a_move_reads_the_moved_rows(dev, size):
    """move_accepted, rope_kv_write and the decode attention one behind the other in a graph, with nothing between them, give what
    they give with a synchronisation after each: the decode kernel asks for the keys of earlier steps before its own wait."""
    from einf_b200 import ops

    heads, kv_heads, page, layers, nodes, cached = 12, 2, 16, 64, 40, [600, 33, 250]
    gen, rng = torch.Generator().manual_seed(size), random.Random(size)
    width = -(-(max(cached) + nodes + 1) // page)
    pages = width * len(cached)
    table = torch.randperm(pages, generator=gen).view(len(cached), width).int().to(dev)
    paths = [[0] + sorted(rng.sample(range(1, nodes), 30)) for _ in cached]
    path, counts, lens = ints(paths, dev), ints([31] * len(cached), dev), ints(cached, dev)
    given = (torch.randn((layers, 2, pages, kv_heads, page, size), generator=gen)).bfloat16().to(dev)
    caches = torch.empty_like(given)
    rows = ops.CacheRows(list(caches.flatten(0, 1).unbind(0)))
    position = ints([c + 31 for c in cached], dev)
    slots = ints([int(table[r, (c + 31) // page]) * page + (c + 31) % page for r, c in enumerate(cached)], dev)
    qkv = torch.randn((len(cached), (heads + 2 * kv_heads) * size), generator=gen).bfloat16().to(dev)
    inv_freq = (100.0 ** (-torch.arange(0, size, 2).float() / size)).to(dev)
    seq, st = ints(range(len(cached)), dev), status(dev)
    q = torch.empty((len(cached), heads, size), dtype=torch.bfloat16, device=dev)
    outs = [torch.zeros_like(q) for _ in range(2 * 3)]

    def step(outs, layers, between):
        caches.copy_(given)
        between()
        ops.move_accepted(rows, table, lens, path, counts, st)
        for out, layer in zip(outs, layers):
            between()
            ops.rope_kv_write(qkv, None, position, inv_freq, slots, q, caches[layer, 0], caches[layer, 1], heads, kv_heads, size, st)
            between()
            ops.paged_decode_attention_tcgen05(q, caches[layer, 0], caches[layer, 1], table, seq, position, out, size ** -0.5, None, 4, st)

    for i, layer in enumerate((0, layers // 2, layers - 1)):
        step(outs[i:i + 1], [layer], torch.cuda.synchronize)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            step(outs[3 + i:4 + i], [layer], lambda: None)
        for _ in range(20):
            outs[3 + i].zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], outs[3 + i])
    assert int(st) == 0


# ---------------------------------------------------------------------------
# Launches cut in the ways that the sizes of tests do not lead to: units over several workers, several units to one, shares that
# the second launch puts together.
def cut_over(monkeypatch, workers):
    from einf_b200 import ops

    def plan(tensor_cores, device, requests, nodes, context, group, kv_heads, size):
        if tensor_cores:
            return "einf_tree_attention_tcgen05", workers, 1, False, ops.TREE_MIN_TILES, 2 * workers * 2 * ops.TREE_TILE, size
        return "einf_tree_attention", workers, 1, False, 1, 2 * workers * ops.TREE_ROWS, -(-size // 4) * 4

    monkeypatch.setattr(ops, "_tree_plan", plan)


class Cut(Trees):
    """Trees that are run several times and stated in 64 bits once."""

    stated: dict = {}

    def check(self, got, window=None, softcap=None):
        key = (window, softcap)
        if key not in self.stated:
            want, bound = ref.tree_attention(self.q, self.k, self.v, self.table, torch.tensor(self.starts), torch.tensor(self.cached),
                                             self.mask, self.scale, self.positions, window, softcap)
            want, bound = want[:self.starts[-1]], bound[:self.starts[-1]]
            if self.q.dtype == torch.bfloat16:      # as in Trees.check
                bound = bound + self.weights_step(window, softcap) + want.abs() * 2.0 ** -8
            self.stated = {**self.stated, key: (want, bound * 1.0001)}
        want, bound = self.stated[key]
        got, live = got.double().cpu(), self.starts[-1]
        assert torch.equal(got[live:], torch.full_like(got[live:], 7.0)), "rows of no request were written"
        assert ((got[:live] - want).abs() <= bound).all()


CUTS = [
    # nodes, cached: one unit, few units, more units than workers
    ([1], [1500]),
    ([40], [1290]),
    ([20, 3, 0, 90, 8], [700, 1500, 40, 300, 900]),
    ([5, 4, 1, 30, 2, 7, 6, 3], [300, 500, 130, 257, 1, 800, 0, 384]),
]


@pytest.mark.parametrize("dtype, heads, kv_heads, size, page", [
    (torch.bfloat16, 14, 2, 64, 16), (torch.bfloat16, 12, 2, 128, 16), (torch.bfloat16, 4, 4, 128, 64), (torch.float32, 4, 2, 48, 4)])
@pytest.mark.parametrize("nodes, cached", CUTS)
def test_tree_attention_cut_over_workers(dev, monkeypatch, dtype, heads, kv_heads, size, page, nodes, cached):
    case = Cut(dev, heads, kv_heads, size, page, nodes, cached, dtype, seed=sum(nodes), extra_rows=1)
    for workers in (1, 2, 3, 7, 148):
        cut_over(monkeypatch, workers)
        first = case.run()
        case.check(first)
        assert torch.equal(first, case.run())


@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("window, softcap", [(200, None), (30, 3.0), (10 ** 9, 20.0)])
def test_windows_and_caps_cut_over_workers(dev, monkeypatch, size, window, softcap):
    case = Cut(dev, 12, 2, size, 16, *CUTS[3], torch.bfloat16, seed=4)
    for workers in (2, 7, 148):
        cut_over(monkeypatch, workers)
        case.check(case.run(window=window, **({"softcap": softcap} if softcap else {})), window, softcap)


@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("levels", [
    lambda j: -100.0 if j < 200 else 150.0 + j % 3, lambda j: 150.0 if j < 200 else -100.0, lambda j: -300.0 - j % 5,
    lambda j: 900.0 if j == 350 else 899.0 if j == 30 else 0.5 * (j % 7)], ids=["rising", "falling", "low", "peaks"])
def test_scores_that_need_a_second_passage_cut_over_workers(dev, monkeypatch, size, levels):
    nodes, cached = CUTS[3]
    case = Cut(dev, 6, 2, size, 16, nodes, cached, torch.bfloat16, seed=6)
    case.q[:] = 1.0
    for r, (c, n) in enumerate(zip(cached, nodes)):
        for j in range(c + n):
            where, row = case.slot(r, j)
            case.k[where, :, row] = levels(j) * size ** -0.5
    for workers in (2, 3, 7, 148):
        cut_over(monkeypatch, workers)
        case.check(case.run())


@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("workers", [2, 7, 148])
@pytest.mark.parametrize("bad", [NAN, math.inf])
def test_values_that_are_not_finite_cut_over_workers(dev, monkeypatch, size, workers, bad):
    cut_over(monkeypatch, workers)
    nodes, cached = CUTS[2]
    case, clean = (Trees(dev, 12, 2, size, 16, nodes, cached, torch.bfloat16, seed=11) for _ in range(2))
    hit = 5
    where, row = case.slot(0, cached[0] + hit)
    case.v[where, 0, row, ::3] = bad
    got, want = case.run().double().cpu(), clean.run().double().cpu()
    for j in range(nodes[0]):
        if int(case.mask[j, 0]) >> hit & 1:
            assert not got[j, :6, ::3].isfinite().any()
            got[j, :6, ::3] = want[j, :6, ::3]
    assert torch.equal(got, want)


@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("workers", [3, 148])
def test_graphs_that_share_scratch_memory_at_once(dev, monkeypatch, size, workers):
    """Two captured launches with shares in scratch memory, replayed side by side, and a third one on another stream meanwhile."""
    from einf_b200 import ops

    cut_over(monkeypatch, workers)
    cases = [Trees(dev, 12, 2, size, 16, *CUTS[i], torch.bfloat16, seed=2 + i) for i in (2, 3, 2)]
    wants, st = [case.run() for case in cases], status(dev)
    given, outs, streams, graphs = [case.arguments() for case in cases], [torch.zeros_like(w) for w in wants], [torch.cuda.Stream() for _ in cases], []
    torch.cuda.synchronize()
    for case, arguments, out in zip(cases[:2], given, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.tree_attention(*arguments, out, case.scale, st)
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            ops.tree_attention(*given[2], outs[2], cases[2].scale, st)
    torch.cuda.synchronize()
    assert int(st) == 0 and all(torch.equal(want, out) for want, out in zip(wants, outs))


@pytest.mark.parametrize("dtype, heads, kv_heads, size, page", [
    (torch.bfloat16, 14, 2, 64, 16), (torch.bfloat16, 6, 2, 128, 8), (torch.bfloat16, 4, 2, 48, 4), (torch.float32, 4, 2, 20, 5)])
@pytest.mark.parametrize("requests", [33, 70])
def test_more_requests_than_a_warp_has_lanes(dev, monkeypatch, dtype, heads, kv_heads, size, page, requests):
    """A launch's work is counted 32 requests at a time; some of them, the last and a whole 32 among them, have no nodes."""
    rng = random.Random(requests)
    nodes = [rng.choice([0, 1, 2, 5]) for _ in range(requests)]
    cached = [rng.choice([0, 1, 30, 127, 128, 300]) for _ in range(requests)]
    nodes[-1] = 0
    if requests > 64:
        nodes[32:64] = [0] * 32
    case = Cut(dev, heads, kv_heads, size, page, nodes, cached, dtype, seed=requests, extra_rows=1)
    for workers in (None, 5, 148):
        if workers:
            cut_over(monkeypatch, workers)
        case.check(case.run())
        case.check(case.run(window=100), 100)


@pytest.mark.parametrize("dtype, heads, size", [(torch.float32, 32, 1), (torch.bfloat16, 128, 64)])
def test_more_tiles_than_a_launch_counts_set_the_status_word(dev, monkeypatch, dtype, heads, size):
    """One page over and over: more than 2^31 pairs of rows' and keys' tiles, in a few hundred megabytes."""
    from einf_b200 import ops

    cut_over(monkeypatch, 148)
    nodes, cached, page = (16384, 1 << 22, 64) if size == 1 else (32768, 1 << 24, 64)
    k = torch.zeros((1, 1, page, size), dtype=dtype, device=dev)
    q = torch.zeros((nodes, heads, size), dtype=dtype, device=dev)
    table = torch.zeros((1, -(-(cached + nodes) // page)), dtype=torch.int32, device=dev)
    out, st = torch.full_like(q, 7.0), status(dev)
    ops.tree_attention(q, k, k.clone(), table, ints([0, nodes], dev), ints([cached], dev), torch.ones((nodes, 1), dtype=torch.int64, device=dev),
                       out, 1.0, st)
    assert int(st) == ops.STATUS_BAD_INDEX
    assert (out == 7.0).all()


def test_trees_that_overlap_to_more_than_their_nodes_set_the_status_word(dev):
    """The same rows for every second request, the launch's most units each: counted in 64 bits, and not computed."""
    from einf_b200 import ops

    nodes, requests = 1 << 20, 8192
    q = torch.zeros((nodes, 1, 1), device=dev)
    k = torch.zeros((1, 1, nodes, 1), device=dev)
    out, st = torch.full_like(q, 7.0), status(dev)
    starts = torch.tensor([0, nodes] * (requests // 2) + [0], dtype=torch.int32, device=dev)
    table = torch.zeros((requests, 1), dtype=torch.int32, device=dev)
    ops.tree_attention(q, k, k.clone(), table, starts, torch.zeros(requests, dtype=torch.int32, device=dev),
                       torch.zeros((nodes, 1), dtype=torch.int64, device=dev), out, 1.0, st)
    assert int(st) == ops.STATUS_BAD_INDEX
    assert (out == 7.0).all()


@pytest.mark.parametrize("dtype, heads, kv_heads, size, page", [
    (torch.float32, 4, 2, 48, 4), (torch.bfloat16, 4, 2, 48, 4), (torch.bfloat16, 14, 2, 64, 16), (torch.bfloat16, 12, 2, 128, 16)])
@pytest.mark.parametrize("softcap", [3.0, 100.0])
@pytest.mark.parametrize("workers", [None, 7])
def test_infinite_scores_are_capped(dev, monkeypatch, dtype, heads, kv_heads, size, page, softcap, workers):
    """A score of minus or plus infinity is the cap's lowest or highest, for rows that see nothing else too; one that is no number
    stays none."""
    if workers:
        cut_over(monkeypatch, workers)
    nodes, cached = [12, 1, 30, 4], [150, 0, 390, 300]
    case = Trees(dev, heads, kv_heads, size, page, nodes, cached, dtype, seed=11)
    case.q[:, :, 1] = case.q[:, :, 1].abs() + 0.5
    key_size = float((case.k[~case.k.isnan()]).abs().max())
    for r, (c, n) in enumerate(zip(cached, nodes)):
        for j in range(c + n):
            where, row = case.slot(r, j)
            if r == 1 or j % 7 == 3 or (r == 3 and j < 256):
                case.k[where, :, row, 1] = -math.inf
            elif j % 31 == 5:
                case.k[where, :, row, 1] = math.inf
    where, row = case.slot(0, cached[0] + 5)
    case.k[where, :, row, 1] = NAN
    got = case.run(softcap=softcap).double().cpu()
    statement = (case.table, torch.tensor(case.starts), torch.tensor(case.cached), case.mask, case.scale, None, None, softcap)
    want, _ = ref.tree_attention(case.q, case.k, case.v, *statement)
    assert torch.equal(got.isnan(), want.isnan()) and want.isnan().any() and want[12].isfinite().all()
    # A finite score is a sum of `size` rounded products, the cap's own error 8 units of the cap; a weight is off by as much
    # and 4 units more, a result by twice the worst of them and a unit for every sum, of the values' size.
    eps, count = 2.0 ** -24, max(c + n for c, n in zip(cached, nodes))
    worst = (size + 4) * eps * key_size * float(case.q.abs().max()) * size * case.scale + 8 * eps * softcap + 4 * eps * (2 * softcap + 1)
    bound = (2 * worst + (2 * count + count / 16 + 8) * eps) * float(case.v[~case.v.isnan()].abs().max())
    if dtype == torch.bfloat16:      # the weights as the second product's operand, and the result
        sizes, _ = ref.tree_attention(case.q, case.k, case.v.abs(), *statement)
        bound = bound + sizes * 2.0 ** -8 * 1.01 + want.abs() * 2.0 ** -8
    assert ((got - want).abs() <= bound)[want.isfinite()].all()


@pytest.mark.parametrize("dtype, heads, kv_heads, size, page", [
    (torch.float32, 4, 2, 48, 4), (torch.bfloat16, 4, 2, 48, 4), (torch.bfloat16, 14, 2, 64, 16), (torch.bfloat16, 12, 2, 128, 16)])
@pytest.mark.parametrize("workers", [None, 1, 2, 7, 148])
def test_rows_whose_scores_are_all_minus_infinity_are_no_numbers(dev, monkeypatch, dtype, heads, kv_heads, size, page, workers):
    """As their softmax: not zeros, which is what a row gets that sees nothing.  Keys with such a score count for nothing beside others,
    wherever a row's shares begin and end."""
    if workers:
        cut_over(monkeypatch, workers)
    nodes, cached = [12, 1, 30, 4, 3, 9], [150, 0, 390, 300, 700, 0]
    case = Trees(dev, heads, kv_heads, size, page, nodes, cached, dtype, seed=12)
    case.q[:, :, 1] = case.q[:, :, 1].abs() + 0.5
    key_size = float((case.k[~case.k.isnan()]).abs().max())
    for r, (c, n) in enumerate(zip(cached, nodes)):
        for j in range(c + n):
            where, row = case.slot(r, j)
            if r in (1, 4) or (r == 0 and j < 140) or (r == 2 and j >= 128) or (r == 3 and not 256 <= j < 260):
                case.k[where, :, row, 1] = -math.inf
    case.mask[50 + 3] = 0      # of the last request, which has no cached tokens: one node sees nothing
    got = case.run().double().cpu()
    statement = (case.table, torch.tensor(case.starts), torch.tensor(case.cached), case.mask, case.scale)
    want, _ = ref.tree_attention(case.q, case.k, case.v, *statement)
    assert torch.equal(got.isnan(), want.isnan())
    assert want[12].isnan().all() and want[47:50].isnan().all() and int(want.isnan().any(-1).any(-1).sum()) == 4
    assert (want[53] == 0).all() and (got[53] == 0).all()
    # as the bound of other rows: a score is a sum of `size` rounded products, a weight is off by as much and by two units of
    # how far it lies below the row's highest
    eps, count = 2.0 ** -24, max(c + n for c, n in zip(cached, nodes))
    highest = key_size * float(case.q.abs().max()) * size * case.scale
    worst = (size + 4) * eps * highest + 2 * eps * 2 * highest + 4 * eps
    bound = (2 * worst + (2 * count + count / 16 + 8) * eps) * float(case.v[~case.v.isnan()].abs().max())
    if dtype == torch.bfloat16:
        sizes, _ = ref.tree_attention(case.q, case.k, case.v.abs(), *statement)
        bound = bound + sizes * 2.0 ** -8 * 1.01 + want.abs() * 2.0 ** -8
    assert ((got - want).abs() <= bound)[want.isfinite()].all()


@pytest.mark.parametrize("dtype, heads, kv_heads, size, page", [
    (torch.float32, 4, 2, 48, 4), (torch.bfloat16, 14, 2, 64, 16), (torch.bfloat16, 12, 2, 128, 16)])
@pytest.mark.parametrize("workers", [None, 7])
@pytest.mark.parametrize("power, level", [(83, 35.0), (83, 26.0), (-83, -35.0), (-83, -26.0)])
def test_large_and_small_values_beside_scores_far_apart(dev, monkeypatch, dtype, heads, kv_heads, size, page, workers, power, level):
    """What weighs a row's keys against the first it sees has room for values of 2^83 times the weights of scores far above, and loses
    nothing of values of 2^-83 times those of scores far below."""
    if workers:
        cut_over(monkeypatch, workers)
    nodes, cached = ([9, 40], [700, 390]) if level > 0 else ([300, 200], [0, 0])
    case = Trees(dev, heads, kv_heads, size, page, nodes, cached, dtype, seed=13)
    case.q[:] = 1.0
    case.v = (case.v.float() * 2.0 ** power).to(dtype)
    for r, (c, n) in enumerate(zip(cached, nodes)):
        for j in range(c + n):
            where, row = case.slot(r, j)
            case.k[where, :, row] = (0.0 if j < 130 else level - j % 3) * size ** -0.5
    if level < 0:       # a node sees itself and one before it: nothing of the first tiles
        for i in range(sum(nodes)):
            k = i % 300
            case.mask[i] = torch.tensor(words_of(1 << k | 1 << max(k - 1, 0), case.mask.shape[1]))
    case.check(case.run())
