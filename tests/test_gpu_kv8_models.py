"""The 8-bit cache behind the decoder layers (gemma.KV8Cache, kernels.KV8Rows): decode steps of the backbone and flow-matching steps of the
expert, the fused runtimes against the reference runtime bit for bit, replays of a captured step, rewinding; and one attention layer's
operators in a row (norm to INT8 rows, W8A8 product, rotary positions, cache, attention) against 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF, FP = torch.bfloat16, torch.float32


@pytest.fixture(scope='module', autouse=True)
def _lib():
    from yanlongvla_amd import _lib
    _lib.lib()
    torch.cuda.init()


def rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).bfloat16()


@pytest.mark.parametrize('runtime', ['fly', 'resident'])
@pytest.mark.parametrize('P', [70, 64, 5])
def test_backbone_decode_steps(runtime, P):
    """Steps on a KV8Cache: the fused layers give the reference runtime's hidden states bit for bit, twice after a rewind, and the cache
    holds the same rows on both, the prefill's within half a code (1 / 254 of the largest key); a full cache refuses another row."""
    from yanlongvla_amd import gemma, kernels, modules
    x = rand(P + 3, 2048, seed=8)
    out = {}
    for rt in ('reference', runtime):
        model = gemma.make_policy(gemma.BackbonePolicy, DEV, seed=5, layers=2, vocab=512)
        modules.install(model, runtime=rt, layers=gemma.synthetic_layers(model, 14, DEV))
        with torch.inference_mode():
            _, ks, vs = model.prefill(x[:P])
            cache = gemma.KV8Cache(ks, vs, 3)
            runs = []
            for _ in range(2):
                cache.rewind()
                runs.append([model.decode_step_cached(x[P + t:P + t + 1], cache).clone() for t in range(3)])
                assert cache.length == P + 3 and int(cache.start) == P + 3
            assert all(torch.equal(a, b) for a, b in zip(*runs))
            with pytest.raises(RuntimeError):
                model.decode_step_cached(x[:1], cache)
            zero = torch.zeros(1, dtype=torch.int32, device=DEV)
            rows = [kernels.kv8_read(c, zero, cache.start, P + 3, FP) for c in cache.caches]
        out[rt] = runs[0], rows
        k16 = ks[0].float()
        assert ((rows[0][0][0, :P, 0] - k16).abs() <= k16.abs().max() / 254 * 1.001).all()
        assert all(torch.isfinite(a).all() for a in runs[0])
    for a, b in zip(out['reference'][0], out[runtime][0]):
        assert torch.equal(a, b)
    for a, b in zip(out['reference'][1], out[runtime][1]):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_captured_decode_step_goes_on():
    """One captured step, replayed: each replay writes the next row and gives the eager step's hidden state."""
    from yanlongvla_amd import gemma, modules
    model = gemma.make_policy(gemma.BackbonePolicy, DEV, seed=5, layers=2, vocab=512)
    modules.install(model, runtime='fly', layers=gemma.synthetic_layers(model, 14, DEV))
    x = rand(80, 2048, seed=9)
    with torch.inference_mode():
        _, ks, vs = model.prefill(x[:62])
        eager, cache = gemma.KV8Cache(ks, vs, 10), gemma.KV8Cache(ks, vs, 10)
        want = [model.decode_step_cached(x[62 + t:63 + t], eager).clone() for t in range(6)]
        tok = x[62:63].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            model.decode_step_cached(tok, cache)
        torch.cuda.current_stream().wait_stream(side)
        cache.rewind()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            h = model.decode_step_cached(tok, cache)
        cache.rewind()
        for t in range(6):
            tok.copy_(x[62 + t:63 + t])
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(h, want[t])


@pytest.mark.parametrize('runtime', ['fly', 'resident'])
def test_expert_steps_replace_their_rows(runtime):
    """Flow-matching steps against an 8-bit prefix: every step's action tokens take the place of the last step's, so a step's result
    depends on its own input alone, and equals the reference runtime's."""
    from yanlongvla_amd import gemma, kernels, modules
    P, M = 90, 50
    cfg = dict(layers=2)
    prefix = [(rand(P, 256, seed=20 + i), rand(P, 256, seed=30 + i)) for i in range(2)]
    noise = [rand(M, 32, seed=40 + i) for i in range(2)]
    out = {}
    for rt in ('reference', runtime):
        model = gemma.make_policy(gemma.ExpertPolicy, DEV, seed=3, **cfg)
        modules.install(model, runtime=rt, layers=gemma.synthetic_layers(model, 6, DEV))
        start = torch.zeros(1, dtype=torch.int32, device=DEV)
        handles = []
        for k, v in prefix:
            c = kernels.kv8_cache(1, 1, 256, P + M, DEV)
            kernels.kv8_append(c, k[:, None], v[:, None], start)
            handles.append(kernels.KV8Rows(c, torch.full_like(start, P)))
        model.set_prefix(handles, [None] * 2)
        with torch.inference_mode():
            out[rt] = [model.velocity(noise[i]).clone() for i in (0, 1, 0)]
        assert torch.equal(out[rt][0], out[rt][2]) and not torch.equal(out[rt][0], out[rt][1])
    assert all(torch.equal(a, b) for a, b in zip(out['reference'], out[runtime]))


def test_layer_of_operators_against_fp64():
    """Two prompts of different lengths, then a step for both, through norm -> INT8 product (q | k | v) -> rotary positions -> cache ->
    attention. The INT8 rows and the product are checked where they are made; from the product's BF16 rows on, everything is held to 64 bits:
    rotary rows to a BF16 step, the cache's values to the definition, the attention to 2^-8 + 2e-4 of its norm."""
    from yanlongvla_amd import kernels as K
    Hq, Hk, D, W = 16, 8, 128, 1024
    N = (Hq + 2 * Hk) * D
    g = torch.Generator(device=DEV).manual_seed(1)
    w = torch.randn(W, generator=g, device=DEV).mul(0.1).bfloat16()
    w8 = torch.randint(-127, 128, (N, W), generator=g, device=DEV).to(torch.int8)
    sw = torch.full((N,), 1.5 / 73 / W ** 0.5, device=DEV)
    freq, axis = K.rope_frequencies(D, 1e6, (24, 20, 20), True, device=DEV)
    cache = K.kv8_cache(2, Hk, D, 300, DEV)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)     # noqa: E731
    held = [[], []]                                                      # rotated keys and the values of each sequence
    start = [0, 0]
    for counts in ([130, 57], [1, 1], [1, 1]):
        rows = sum(counts)
        x, r = rand(rows, W, seed=50 + start[0]), rand(rows, W, seed=90 + start[0])
        q8, s = torch.empty(rows, W, dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
        K.add_norm_quantize(x, r, w, 1e-6, q8, s, r)
        y = torch.empty(rows, N, dtype=BF, device=DEV)
        K.gemm_i8(q8, w8, y, sa=s, sw=sw)
        want = (q8.double() @ w8.double().t()) * s.double()[:, None] * sw.double()
        assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-6).all()
        q, k, v = (t.unflatten(1, (-1, D)) for t in y.split([Hq * D, Hk * D, Hk * D], 1))
        pos = torch.cat([torch.stack([torch.arange(st, st + n), torch.arange(n) // 8 + st, torch.arange(n) % 8 + st]) for st, n in zip(start, counts)], 1).to(DEV)
        a = (pos[axis.long()].double() * freq[:, None]).t()[:, None]
        turned = []
        for t in (q, k):
            f = t.double()
            lo, hi = f[..., :D // 2], f[..., D // 2:]
            turned.append(torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1))
        K.rope_axes(q, k, pos, freq, axis)                               # in place, views of the product's rows
        for t, z in zip((q, k), turned):
            assert ((t.double() - z).abs() <= 2.0 ** -8 * z.abs() + 1e-5).all()
        cu = ints([0, counts[0], rows])
        K.kv8_append(cache, k, v, ints(start), cu, max(counts))
        lens = [st + n for st, n in zip(start, counts)]
        o = K.kv8_attend(q, cache, ints(lens), cu=cu, most=max(counts))
        kk, vv = K.kv8_read(cache, ints([0, 0]), ints(lens), max(lens), FP)
        at = 0
        for b, n in enumerate(counts):
            held[b].append((k[at:at + n], v[at:at + n]))
            for got, i in ((kk, 0), (vv, 1)):
                full = torch.cat([h[i] for h in held[b]]).float()
                for j in range(0, lens[b], 64):                         # off by at most half a code of the block's largest value
                    part = full[j:j + 64]
                    big = part.abs().amax((0, 2))[None, :, None]
                    assert ((got[b, j:j + len(part)] - part).abs() <= big / 254 * 1.00001).all()
            for h in range(Hq):
                sc = q[at:at + n, h].double() @ kk[b, :lens[b], h // 2].double().t() / D ** 0.5
                sc = sc.masked_fill(torch.arange(lens[b], device=DEV)[None] > torch.arange(n, device=DEV)[:, None] + start[b], float('-inf'))
                ref = torch.softmax(sc, 1) @ vv[b, :lens[b], h // 2].double()
                assert (o[at:at + n, h].double() - ref).norm() <= (2.0 ** -8 + 2e-4) * ref.norm()
            at += n
        start = lens
