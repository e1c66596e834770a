"""GPU tests of a pool's bookkeeping (room, forks, cuts, compaction, copies): every table, length, count, free page and row of the pool against
a model of the definitions in plain Python, over made-up histories, and what calls cannot do; and the cache in pages behind the decoder layers."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope='module', autouse=True)
def _lib():
    from yanlongvla_amd import _lib
    _lib.lib()
    torch.cuda.init()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Model:
    """The definitions, one sequence and page after the other. Pages hold the rows' names (None: never written)."""

    def __init__(self, B, N, pages, T):
        self.B, self.N, self.T = B, N, T
        self.table = [[] for _ in range(B)]
        self.lens = [0] * B
        self.refs = [0] * pages
        self.pool = [[None] * T for _ in range(pages)]
        self.lack = 0

    def held(self, n):
        return -(-n // self.T)

    def drop(self, p):
        self.refs[p] -= 1

    def take(self, more):
        start = list(self.lens)
        spare = [p for p, r in enumerate(self.refs) if not r]
        shared = [r > 1 for r in self.refs]
        used, dropped = 0, []
        for b, m in enumerate(more):
            if m <= 0:
                continue
            if self.lens[b] + m > self.N * self.T:
                self.lack += 1
                continue
            have = self.held(self.lens[b])
            copy = self.lens[b] % self.T != 0 and shared[self.table[b][-1]]
            need = self.held(self.lens[b] + m) - have + copy
            used += need
            if need and used > len(spare):
                self.lack += 1
                continue
            mine = spare[used - need:used]
            if copy:
                old = self.table[b].pop()
                self.pool[mine[0]] = list(self.pool[old])
                dropped.append(old)
            self.table[b] += mine
            for p in mine:
                self.refs[p] = 1
            self.lens[b] += m
        for p in dropped:
            self.drop(p)
        return start

    def write(self, b, start, names):
        for i, name in enumerate(names):
            if start + i < self.lens[b]:
                self.pool[self.table[b][(start + i) // self.T]][(start + i) % self.T] = name

    def fork(self, src, dst):
        before = list(self.lens)
        for i, (s, d) in enumerate(zip(src, dst)):
            ok = 0 <= s < self.B and 0 <= d < self.B and s != d and before[d] == 0 and d not in dst[:i] and s not in dst
            if not ok:
                self.lack += 1
                continue
            self.table[d], self.lens[d] = list(self.table[s]), self.lens[s]
            for p in self.table[d]:
                self.refs[p] += 1

    def trim(self, keep):
        for b, n in enumerate(keep):
            self.lens[b] = max(0, min(self.lens[b], n))
            while len(self.table[b]) > self.held(self.lens[b]):
                self.drop(self.table[b].pop())

    def compact(self):
        U = sum(r > 0 for r in self.refs)
        high = [p for p, r in enumerate(self.refs) if r and p >= U]
        low = [p for p, r in enumerate(self.refs) if not r and p < U]
        to = dict(zip(high, low))
        for s, d in to.items():
            self.refs[s], self.refs[d] = 0, self.refs[s]
            self.pool[d] = list(self.pool[s])
        self.table = [[to.get(p, p) for p in t] for t in self.table]


def compare(pt, pool, m):
    table = [t + [-1] * (m.N - len(t)) for t in m.table]
    assert pt.table.tolist() == table
    assert pt.lens.tolist() == m.lens and pt.refs.tolist() == m.refs and pt.lack.item() == m.lack
    bits = [w & 0xffffffff for w in pt.free.tolist()]
    assert [(bits[p // 32] >> (p % 32)) & 1 for p in range(len(m.refs))] == [int(r == 0) for r in m.refs]
    assert sum(bin(w).count('1') for w in bits) == sum(r == 0 for r in m.refs)
    names = torch.tensor([[-1.0 if x is None else x for x in page] for page in m.pool])
    used = torch.tensor([r > 0 for r in m.refs])
    for l in range(pool.k.shape[0]):
        k, v = pool.k[l].float().cpu(), pool.v[l].float().cpu()
        assert (k == k[:, :1, :, :1]).all() and (v == v[:, :1, :, :1]).all()
        have = used[:, None] & (names >= 0)
        assert torch.equal(k[:, 0, :, 0][have], names[have] + l) and torch.equal(v[:, 0, :, 0][have], names[have] + l + 64)


@pytest.mark.parametrize('seed', range(12))
def test_made_up_histories(seed):
    """Random calls, at times beyond what the pool or a sequence holds, with pairs that cannot be forked; rows are named by whole numbers that BF16 holds."""
    from yanlongvla_amd import kernels as K
    rng = random.Random(seed)
    B, T = rng.choice((1, 3, 8, 33)), rng.choice((16, 32, 64))
    N, P, L, H, D = rng.randint(1, 6), rng.choice((1, 7, 32, 33, 70)), 2, rng.choice((1, 3)), rng.choice((8, 64))
    pool, pt, m = K.kv_pages(P, H, D, DEV, T, layers=L), K.page_table(B, N, P, DEV, T), Model(B, N, P, T)
    for _ in range(25):
        kind = rng.choice(('take', 'take', 'take', 'fork', 'trim', 'compact'))
        if kind == 'take':
            more = [rng.choice((0, 0, 1, rng.randint(1, 2 * T), rng.randint(1, N * T))) for _ in range(B)]
            start = K.pages_take(pt, pool, ints(more))
            assert start.tolist() == m.take(more)
            names = [[float(rng.randint(0, 60)) for _ in range(n)] for n in more]
            rows = torch.tensor([x for r in names for x in r], device=DEV)[:, None, None].expand(-1, H, D).to(BF)
            cu = ints([sum(more[:b]) for b in range(B + 1)])
            for l in range(L):
                K.paged_append(K.Pages(pool.k[l], pool.v[l]), rows + l, rows + l + 64, pt.table, pt.lens, start, cu, max(max(more), 1))
            for b in range(B):
                m.write(b, start[b].item(), names[b])
        elif kind == 'fork':
            n = rng.randint(1, 4)
            src, dst = ([rng.randint(-1, B) if rng.random() < 0.2 else rng.randrange(B) for _ in range(n)] for _ in range(2))
            K.pages_fork(pt, ints(src), ints(dst))
            m.fork(src, dst)
        elif kind == 'trim':
            keep = [rng.choice((0, 10 ** 9, rng.randint(-3, N * T))) for _ in range(B)]
            K.pages_trim(pt, ints(keep))
            m.trim(keep)
        else:
            K.pages_compact(pt, pool)
            m.compact()
        compare(pt, pool, m)


def test_many_sequences_and_pages():
    """The most sequences of one table, over several sweeps of the plan's threads, out of more pages than one sweep sees."""
    from yanlongvla_amd import kernels as K
    B, T, P = 4096, 16, 40000
    pool, pt, m = K.kv_pages(P, 1, 8, DEV, T, layers=1), K.page_table(B, 12, P, DEV, T), Model(B, 12, P, T)
    rng = random.Random(0)
    for r in range(3):
        more = [rng.randint(0, 60) for _ in range(B)]
        assert K.pages_take(pt, pool, ints(more)).tolist() == m.take(more)
        keep = [rng.choice((0, 10 ** 6, rng.randint(0, 120))) for _ in range(B)]
        K.pages_trim(pt, ints(keep))
        m.trim(keep)
        K.pages_compact(pt, pool)
        m.compact()
        compare(pt, pool, m)
    src = [b for b in range(B) if m.lens[b]][:500]
    dst = [b for b in range(B) if not m.lens[b]][:500]
    n = min(len(src), len(dst))
    K.pages_fork(pt, ints(src[:n]), ints(dst[:n]))
    m.fork(src[:n], dst[:n])
    more = [60] * B                                                            # more than there is: the first sequences are served
    assert K.pages_take(pt, pool, ints(more)).tolist() == m.take(more)
    compare(pt, pool, m)
    assert m.lack > 0


@pytest.mark.parametrize('dt', [BF, HF])
@pytest.mark.parametrize('layers', [None, 3])
def test_copy(layers, dt):
    from yanlongvla_amd import kernels as K
    pool = K.kv_pages(40, 3, 72, DEV, 16, dt, layers)
    for i, t in enumerate(pool):
        t.copy_(torch.randn(t.shape, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV))
    want = [t.clone() for t in pool]
    src, dst = [1, 5, 1, 39, -1, 3, 7, 40], [2, 0, 38, 20, 4, 40, 7, 9]
    K.pages_copy(pool, ints(src), ints(dst))
    for t in want:
        x = t if layers else t[None]
        for s, d in zip(src, dst):
            if 0 <= s < 40 and 0 <= d < 40:
                x[:, d] = x[:, s].clone()
    assert all(torch.equal(a, b) for a, b in zip(pool, want))
    K.pages_copy(pool, ints([]), ints([]))


def test_captured_bookkeeping():
    """Fork, room, cut and compaction in one graph, replayed: every replay gives what eager calls on the same state give."""
    from yanlongvla_amd import kernels as K
    B, N, P, T = 6, 8, 60, 16
    pool, pt = K.kv_pages(P, 1, 64, DEV, T, layers=2), K.page_table(B, N, P, DEV, T)
    pool2, pt2 = K.kv_pages(P, 1, 64, DEV, T, layers=2), K.page_table(B, N, P, DEV, T)
    first, src, dst, more, keep = ints([50, 20, 0, 0, 0, 0]), ints([0, 1, 0]), ints([2, 3, 4]), ints([1, 2, 30, 4, 5, 0]), ints([9999, 9999, 0, 9999, 0, 0])
    end = ints([45, 0, 0, 0, 0, 0])

    def calls(pt, pool):
        K.pages_take(pt, pool, first)
        K.pages_fork(pt, src, dst)
        start = K.pages_take(pt, pool, more)
        K.pages_trim(pt, keep)
        K.pages_compact(pt, pool)
        seen = torch.cat([pt.table.flatten(), pt.lens, pt.refs, pt.free, start])
        K.pages_trim(pt, end)
        return seen

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls(pt, pool)
    torch.cuda.current_stream().wait_stream(side)
    zero = torch.zeros(B, dtype=torch.int32, device=DEV)
    K.pages_trim(pt, zero)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls(pt, pool)
    for _ in range(4):
        want = calls(pt2, pool2)
        graph.replay()
        assert torch.equal(out, want)
        K.pages_trim(pt2, ints([30, 0, 0, 0, 0, 0]))
        K.pages_trim(pt, ints([30, 0, 0, 0, 0, 0]))
        torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------------- behind the decoder layers
def rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).bfloat16()


@pytest.mark.parametrize('runtime', ['fly', 'resident'])
def test_backbone_decode_steps(runtime):
    """A batch of sequences in pages: the fused layers give the reference runtime's hidden states bit for bit, each sequence alone gives those of
    KVCache within the attentions' rounding, and a fork goes on as its origin would."""
    from yanlongvla_amd import gemma, modules
    lens, steps = [70, 5, 128], 3
    x = [rand(n + steps, 2048, seed=20 + i) for i, n in enumerate(lens)]
    out = {}
    for rt in ('reference', runtime):
        model = gemma.make_policy(gemma.BackbonePolicy, DEV, seed=5, layers=2, vocab=512)
        modules.install(model, runtime=rt, layers=gemma.synthetic_layers(model, 14, DEV))
        with torch.inference_mode():
            cache = gemma.PagedKVCache(2, 4, 30, 256, DEV, rows=16)
            alone = []
            for b, n in enumerate(lens):
                _, ks, vs = model.prefill(x[b][:n])
                cache.extend(ks, vs, b)
                single = gemma.KVCache(ks, vs, steps)
                alone.append([model.decode_step_cached(x[b][n + t:n + t + 1], single).clone() for t in range(steps)])
            cache.active.copy_(ints([1, 1, 1, 0]))
            cache.fork(ints([0]), ints([3]))
            got = [model.decode_step_cached(torch.cat([x[b][n + t:n + t + 1] for b, n in enumerate(lens)] + [x[0][:1]]), cache).clone() for t in range(steps)]
            assert cache.table.lens.tolist() == [73, 8, 131, 70] and cache.table.lack.item() == 0
            cache.trim(ints([0, 8, 131, 70]))                                  # the origin ends, its fork takes the same tokens
            cache.compact()
            cache.active.copy_(ints([0, 0, 0, 1]))
            rows = torch.zeros(4, 2048, dtype=BF, device=DEV)
            again = []
            for t in range(steps):
                rows[3] = x[0][70 + t]
                again.append(model.decode_step_cached(rows, cache)[3].clone())
        out[rt] = got
        for t in range(steps):
            assert torch.equal(again[t], got[t][0])
            for b in range(3):
                a, w = got[t][b].float(), alone[b][t][0].float()
                assert float((a - w).norm() / w.norm()) < 0.03
    assert all(torch.equal(a, b) for a, b in zip(out['reference'], out[runtime]))


def test_prefill_in_chunks():
    """Parts of a prompt behind each other: the rows in the pages and the hidden states are those of one call, as far as the order of sums allows."""
    from yanlongvla_amd import gemma, modules
    model = gemma.make_policy(gemma.BackbonePolicy, DEV, seed=5, layers=2, vocab=512)
    modules.install(model, runtime='fly', layers=gemma.synthetic_layers(model, 14, DEV))
    x = rand(300, 2048, seed=3)
    with torch.inference_mode():
        one, parts = (gemma.PagedKVCache(2, 2, 40, 256, DEV, rows=32) for _ in range(2))
        whole = model.prefill_chunk(x, one, 1)
        got = torch.cat([model.prefill_chunk(p, parts, 1) for p in x.split([130, 1, 64, 105])])
    assert one.table.lens.tolist() == parts.table.lens.tolist() == [0, 300]
    assert float((got.float() - whole.float()).norm() / whole.float().norm()) < 0.03
    _, ks, vs = model.prefill(x)
    first = [int(p) for p in one.table.table[1] if p >= 0]
    k = torch.cat([one.layers[0].k[p, 0] for p in first])[:300]
    assert torch.equal(k, ks[0])                                               # the first layer's rows do not depend on attention
    assert float((whole.float() - model.prefill(x)[0].float()).norm() / whole.float().norm()) < 0.03


def test_expert_denoising_steps_of_several_sequences():
    """Action tokens of a batch, replaced in the pages at every step, against each sequence alone with its prefix tensors."""
    from yanlongvla_amd import gemma, modules
    model = gemma.make_policy(gemma.ExpertPolicy, DEV, seed=6, layers=2)
    modules.install(model, runtime='fly', layers=gemma.synthetic_layers(model, 15, DEV))
    B, M, lens = 3, 50, [100, 64, 33]
    noise = rand(B * M, 32, seed=1)
    with torch.inference_mode():
        cache = gemma.PagedKVCache(2, B, 30, 256, DEV, rows=16)
        alone = []
        for b, n in enumerate(lens):
            ks, vs = ([rand(n, 256, seed=30 * b + i + o) for i in range(2)] for o in (0, 10))
            cache.extend(ks, vs, b)
            model.set_prefix(ks, vs)
            alone.append(model.sample_chunk(noise[b * M:(b + 1) * M], 4))
        layers = cache.take(ints([M] * B))
        model.set_prefix(layers, [None] * 2)
        got = [model.sample_chunk(noise, 4).clone() for _ in range(2)]
    assert torch.equal(*got)
    want = torch.cat(alone).float()
    assert float((got[0].float() - want).norm() / want.norm()) < 0.03
    assert cache.table.lens.tolist() == [n + M for n in lens]
