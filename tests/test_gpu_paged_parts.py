"""GPU tests of attentions whose keys are split into parts, of calls whose last sequences have no rows (their offset is the number of rows, where the
workspace ends). Tolerances as in test_gpu_paged.py."""
import pytest
import torch

from test_gpu_paged import BF, DEV, Pool, check, cross_check, ints, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module', autouse=True)
def _lib():
    from yanlongvla_amd import _lib
    _lib.lib()
    torch.cuda.init()


def parts(name, rows, most, B, Hq, H, D, keys):
    """The parts of a call, by its workspace."""
    from yanlongvla_amd import _lib
    return getattr(_lib.lib(), name)(rows, most, B, Hq, H, D, keys) // (rows * Hq * (D + 2)) or 1


def offsets(new):
    return ints([sum(new[:b]) for b in range(len(new) + 1)])


# (lengths, new rows, Hq, H, D, the least and the most parts: one, four and sixteen waves of the join a row)
LAST = [([400, 70, 33], [1, 0, 0], 8, 1, 256, 2, 8), ([40, 1200, 0], [0, 2, 0], 4, 1, 128, 9, 32), ([6000, 7], [1, 0], 8, 1, 128, 33, 128),
        ([5000, 64, 1], [200, 0, 0], 2, 1, 64, 33, 128), ([900, 900, 5], [150, 130, 0], 4, 2, 128, 2, 8)]


@pytest.mark.parametrize('lens,new,Hq,H,D,least,greatest', LAST)
def test_sequences_without_rows_last(lens, new, Hq, H, D, least, greatest):
    from yanlongvla_amd import _lib, kernels as K
    T, rows, most, keys, B = 16, sum(new), max(new), max(lens), len(lens)
    assert least <= parts('tcq_paged_attend_floats', rows, most, B, Hq, H, D, keys) <= greatest
    pool = Pool(lens, H, D, T, BF, seed=D)
    q, cu = rand(rows, Hq, D, seed=4, by=2.0), offsets(new)
    got = K.paged_attend(q, pool.pages, pool.table, pool.lens, cu=cu, most=most, keys=keys)
    check(got, q, pool, lens, new, True, BF)
    # a workspace of the stated size, and what lies behind it: neither changed nor used
    n = _lib.lib().tcq_paged_attend_floats(rows, most, B, Hq, H, D, keys)
    work = torch.full((n + 1024,), float('nan'), device=DEV)
    o, (k, v) = torch.empty_like(q), pool.pages
    rc = _lib.lib().tcq_paged_attend(q.data_ptr(), *q.stride()[:2], K.DTYPE[BF], cu.data_ptr(), pool.lens.data_ptr(), rows, most, B, Hq, H, D, k.data_ptr(),
                                     *k.stride()[:3], v.data_ptr(), *v.stride()[:3], k.shape[0], T, pool.table.data_ptr(), pool.table.shape[1], 1,
                                     D ** -0.5, keys, work.data_ptr(), o.data_ptr(), K.stream())
    assert rc == 0 and torch.equal(o, got) and work[n:].isnan().all()


def test_cross_attention_of_sequences_without_rows_last():
    from yanlongvla_amd import kernels as K
    B, T, Hq, H, D, new = 3, 1500, 8, 2, 128, [5, 0, 0]
    assert parts('tcq_cross_attend_floats', 5, 5, B, Hq, H, D, T) > 1
    q, k, v = rand(5, Hq, D, seed=1, by=2.0), rand(B, T, H, D, seed=2), rand(B, T, H, D, seed=3)
    got = K.cross_attend(q, k, v, cu=offsets(new), most=5)
    cross_check(got, q, k[:1], v[:1], [T], None, 5, BF)


def test_prefill_chunks_of_sequences_in_turn():
    """Parts of two prompts, behind each other and in turn, in a cache whose other sequences have no rows in a call, its capacity so long that the keys are split."""
    from yanlongvla_amd import gemma, modules
    model = gemma.make_policy(gemma.BackbonePolicy, DEV, seed=5, layers=2, vocab=512)
    modules.install(model, runtime='fly', layers=gemma.synthetic_layers(model, 14, DEV))
    prompts = [rand(n, 2048, seed=n) for n in (150, 97)]
    sizes = [(64, 50, 36), (1, 64, 32)]
    assert parts('tcq_paged_attend_floats', 50, 50, 4, 8, 1, 256, 600 * 16) > 1
    with torch.inference_mode():
        cache = gemma.PagedKVCache(2, 4, 600, 256, DEV, rows=16)
        got = [[], []]
        for i in range(3):
            for b, (x, n) in enumerate(zip(prompts, sizes)):
                at = sum(n[:i])
                got[b].append(model.prefill_chunk(x[at:at + n[i]], cache, 2 * b))
        assert cache.table.lens.tolist() == [150, 0, 97, 0] and cache.table.lack.item() == 0
        for x, h in zip(prompts, got):
            want = model.prefill(x)[0].float()
            assert float((torch.cat(h).float() - want).norm() / want.norm()) < 0.03
