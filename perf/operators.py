"""The attention half of an INT8 decoder layer between its products, as cases that can be timed and compared.

  rope    kernels.rope_axes: rotary positions with one or several axes (time, height, width) on the query and key heads
  append  kernels.kv8_append + kv8_read: new key / value rows into a cache held in 8 bits (one scale for every block of 64
          tokens of a KV head), and the rows of the blocks it touched read back
  attend  kernels.kv8_attend: grouped-query attention of a batch of sequences over that cache
  norm    kernels.add_norm_quantize: residual addition, RMSNorm and INT8 rows with a scale for each token

The plain forms are elementary torch operations in 32 bits (64 for the rotary angles) on the same tensors. The cache's layout is
part of its interface: K codes of a block as (4, D / 16, 16, 16) = (token / 16, dim / 16, token % 16, dim % 16); V codes as
(D / 16, 4, 16, 16) = (dim / 16, token % 16 / 4, dim % 16, token / 16 * 4 + token % 4); scales (K, V) per block; the 16-bit rows
of the newest two blocks as (block % 2, K or V, token, dim).
"""
import math

import torch

own = False
DEV = 'cuda'
T = 64                                                                     # tokens per cache block
DT = dict(bf16=torch.bfloat16, f16=torch.float16, f32=torch.float32)


def listed():
    return [
        # one generated token of a language model with image positions: the fewest bytes, latency only
        dict(name='rope_token', kind='rope', M=1, Hq=16, Hk=8, D=128, R=128, axes=3, far=4000, dtype='bf16', inverse=False),
        # a prompt of several images and its text
        dict(name='rope_prompt', kind='rope', M=2048, Hq=16, Hk=8, D=128, R=128, axes=3, far=3000, dtype='bf16', inverse=False),
        # the gradient of a vision tower's 2-D positions, in FP32, patch count odd
        dict(name='rope_vision_grad', kind='rope', M=4761, Hq=16, Hk=16, D=64, R=64, axes=2, far=69, dtype='f32', inverse=True),
        # a decode step of a batch of sequences: one row each into a block that is partly filled
        dict(name='append_step', kind='append', B=16, M=1, P=1000, H=1, D=256, ragged=True, dtype='bf16'),
        # prompts of different lengths behind what a cache holds already
        dict(name='append_prompt', kind='append', B=6, M=1000, P=777, H=8, D=128, ragged=True, dtype='bf16'),
        # one generated token behind the prefix of one observation
        dict(name='attend_token', kind='attend', B=1, M=1, P=968, Hq=8, Hk=1, D=256, causal=True, ragged=False, dtype='bf16'),
        # a decode step of a batch, grouped heads, lengths between 4 and 8 thousand
        dict(name='attend_batch', kind='attend', B=16, M=1, P=8192, Hq=16, Hk=8, D=128, causal=True, ragged=True, dtype='bf16'),
        # a generated token behind very long contexts
        dict(name='attend_long', kind='attend', B=2, M=1, P=131000, Hq=8, Hk=1, D=256, causal=True, ragged=True, dtype='f16'),
        # the action tokens of several robots: every token sees the prefix and all action tokens
        dict(name='attend_actions', kind='attend', B=4, M=50, P=800, Hq=8, Hk=1, D=256, causal=False, ragged=False, dtype='bf16'),
        # a part of a long prompt behind the parts before it
        dict(name='attend_prompt', kind='attend', B=2, M=1024, P=4096, Hq=16, Hk=8, D=128, causal=True, ragged=True, dtype='bf16'),
        # one token's residual stream
        dict(name='norm_token', kind='norm', M=1, K=2048, dtype='bf16', offset=1.0),
        # a batch of prompts at the widest hidden size
        dict(name='norm_prompt', kind='norm', M=4000, K=4096, dtype='bf16', offset=0.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(('rope', 'append', 'attend', 'attend', 'norm'))
    if kind == 'rope':
        D = rng.choice((64, 128, 256))
        Hk = _log_int(rng, 1, 16)
        M = _log_int(rng, 1, 4096 * 128 // D // (1 + Hk // 4))
        return dict(kind='rope', M=M, Hq=Hk * rng.randint(1, 2), Hk=Hk, D=D, R=rng.choice((D, D // 2)), axes=rng.randint(1, 3),
                    far=_log_int(rng, 10, 100000), dtype=rng.choice(('bf16', 'f16', 'f32')), inverse=rng.random() < 0.3)
    if kind == 'append':
        H, D = rng.choice(((1, 256), (1, 128), (2, 64), (4, 128), (8, 128), (8, 64)))
        B = rng.randint(1, 8)
        return dict(kind='append', B=B, M=_log_int(rng, 1, 4000 // B), P=rng.randint(0, 2000), H=H, D=D, ragged=rng.random() < 0.6,
                    dtype=rng.choice(('bf16', 'f16')))
    if kind == 'norm':
        K = rng.choice((1024, 1152, 1536, 2048, 2560, 4096, 4304, 6144, 8192, 16384, 16 * rng.randint(4, 512)))
        return dict(kind='norm', M=_log_int(rng, 1, 16000000 // K), K=K, dtype=rng.choice(('bf16', 'f16')), offset=rng.choice((0.0, 1.0)))
    most = work(listed()[9])
    while True:
        Hk, G, D = rng.choice(((1, 8, 256), (1, 5, 256), (8, 2, 128), (2, 7, 128), (4, 4, 64), (16, 1, 64), (1, 16, 128)))
        M = 1 if rng.random() < 0.4 else _log_int(rng, 1, 1500)
        case = dict(kind='attend', B=_log_int(rng, 1, 32), M=M, P=_log_int(rng, 1, 120000) - 1, Hq=Hk * G, Hk=Hk, D=D,
                    causal=rng.random() < 0.8, ragged=rng.random() < 0.6, dtype=rng.choice(('bf16', 'f16')))
        w = work(case)
        if w['flops'] <= most['flops'] and w['bytes'] <= 1.5e8 and M * case['B'] * case['Hq'] * (case['P'] + M) <= 4e8:
            return case


def _counts(case):
    """Rows that B sequences hold and new rows, the first sequence's M behind P and, ragged, the others' down to half of it. What
    appends more than a block starts at a block, so that a pass can be made again on the same cache: the rows that it
    starts from are still those of the newest blocks."""
    B = case['B']
    start, new = ([n - (b * n) // (2 * B) if case['ragged'] else n for b in range(B)] for n in (case['P'], case['M']))
    return [s // T * T if n > T and case['kind'] == 'append' else s for s, n in zip(start, new)], new


# ---------------------------------------------------------------------------------------------------------------- prepare
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DT[case['dtype']]
    st = dict(case=case)
    if case['kind'] == 'rope':
        M, D, R, A = case['M'], case['D'], case['R'], case['axes']
        st['q'] = torch.randn(M, case['Hq'], D, generator=g, device=DEV).to(dt)
        st['k'] = torch.randn(M, case['Hk'], D, generator=g, device=DEV).to(dt)
        st['pos'] = torch.randint(0, case['far'] + 1, (A, M), generator=g, device=DEV, dtype=torch.int32)
        st['freq'] = 10000.0 ** (-torch.arange(R // 2, device=DEV, dtype=torch.float64) / (R // 2))
        st['axis'] = torch.arange(R // 2, device=DEV, dtype=torch.int32) % A
        return st
    if case['kind'] == 'norm':
        M, K = case['M'], case['K']
        wide = torch.randn(K, generator=g, device=DEV).mul(0.7).exp()               # some columns carry far larger values
        st['x'] = torch.randn(M, K, generator=g, device=DEV).to(dt)
        st['r'] = (torch.randn(M, K, generator=g, device=DEV) * wide).to(dt)
        st['w'] = (torch.randn(K, generator=g, device=DEV) * 0.2 + 1 - case['offset']).to(dt)
        return st
    B, M, D, H = case['B'], case['M'], case['D'], case.get('H', case.get('Hk'))
    start, new = _counts(case)
    nblk = max(s + n for s, n in zip(start, new)) // T + 1
    cum = [sum(new[:b]) for b in range(B + 1)]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)                 # noqa: E731
    st.update(start=ints(start), lens=ints([s + n for s, n in zip(start, new)]), cu=ints(cum), most=max(new),
              first=ints([s // T * T for s in start]), rows=(M + T - 1 + T - 1) // T * T)

    def codes(*shape):
        return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * 30).round_().clamp_(-127, 127).to(torch.int8)

    st['k8'] = codes(B, H, nblk, 4, D // 16, 16, 16)
    st['v8'] = codes(B, H, nblk, D // 16, 4, 16, 16)
    st['scale'] = (torch.rand(B, H, nblk, 2, generator=g, device=DEV) + 0.5) / 30
    st['tail'] = torch.randn(B, H, 2, 2, T, D, generator=g, device=DEV).to(dt)
    if case['kind'] == 'append':
        st['k'] = torch.randn(cum[-1], H, D, generator=g, device=DEV).to(dt)
        st['v'] = torch.randn(cum[-1], H, D, generator=g, device=DEV).to(dt)
    else:
        st['q'] = (torch.randn(cum[-1], case['Hq'], D, generator=g, device=DEV) * 2).to(dt)
    return st


# -------------------------------------------------------------------------------------------------------------------- run
def run(st):
    case = st['case']
    kind = case['kind']
    if own:
        from yanlongvla_amd import kernels
        if kind == 'rope':
            q, k = torch.empty_like(st['q']), torch.empty_like(st['k'])
            kernels.rope_axes(st['q'], st['k'], st['pos'], st['freq'], st['axis'], q, k, inverse=case['inverse'])
            return dict(q=q, k=k)
        if kind == 'norm':
            x = st['x']
            h, q = torch.empty_like(x), torch.empty_like(x, dtype=torch.int8)
            scale = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
            kernels.add_norm_quantize(x, st['r'], st['w'], 1e-6, q, scale, h, offset=case['offset'])
            return dict(sum=h, scale=scale, values=torch.mul(q, scale[:, None], out=torch.empty_like(x)))
        cache = kernels.KV8(st['k8'], st['v8'], st['scale'], st['tail'])
        if kind == 'append':
            kernels.kv8_append(cache, st['k'], st['v'], st['start'], st['cu'], st['most'])
            k, v = kernels.kv8_read(cache, st['first'], st['lens'], st['rows'])
            return dict(k=k, v=v, tail=st['tail'])
        return kernels.kv8_attend(st['q'], cache, st['lens'], causal=case['causal'], cu=st['cu'], most=st['most'])
    if kind == 'rope':
        return dict(zip('qk', _rope(st)))
    if kind == 'norm':
        return _norm(st)
    return _append(st) if kind == 'append' else _attend(st)


def _rope(st):
    case = st['case']
    half = case['R'] // 2
    angle = st['pos'][st['axis'].long()].t().double() * st['freq']                   # (M, R / 2)
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    s = -s if case['inverse'] else s
    out = []
    for x in (st['q'], st['k']):
        a, b, rest = x[..., :half].float(), x[..., half:2 * half].float(), x[..., 2 * half:]
        out.append(torch.cat([(a * c - b * s).to(x.dtype), (b * c + a * s).to(x.dtype), rest], -1))
    return out


def _norm(st):
    x, w = st['x'], st['w']
    h = (x.float() + st['r'].float()).to(x.dtype)
    f = h.float()
    n = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6) * (st['case']['offset'] + w.float())
    big = n.abs().amax(-1, keepdim=True)
    scale = torch.where(big > 0, big / 127, torch.ones_like(big))
    return dict(sum=h, scale=scale[:, 0], values=((n / scale).round().clamp(-127, 127) * scale).to(x.dtype))


def _owners(st):
    """Sequence and place of every new row."""
    r = torch.arange(int(st['q' if 'q' in st else 'k'].shape[0]), device=DEV)
    b = torch.searchsorted(st['cu'].long(), r, right=True) - 1
    return b, r - st['cu'].long()[b]


def _append(st):
    case, tail = st['case'], st['tail']
    B, H, D, n = case['B'], case['H'], case['D'], st['rows']
    start, end = st['start'].long()[:, None], st['lens'].long()[:, None]
    new = torch.stack([st['k'], st['v']])                                            # (2, rows, H, D)
    # the rows of the touched blocks: 16-bit rows kept of the first one, then the new rows, then nothing
    at = st['first'].long()[:, None] + torch.arange(n, device=DEV)                  # (B, n) positions
    src = (st['cu'].long()[:-1, None] + at - start).clamp(0, new.shape[1] - 1)
    fresh = new[:, src].permute(1, 3, 0, 2, 4).float()                               # (B, H, 2, n, D)
    b = torch.arange(B, device=DEV)[:, None]
    kept = tail[b, :, at // T % 2, :, at % T].permute(0, 2, 3, 1, 4).float()
    at5, start5, end5 = (t[:, None, None, :, None] for t in (at, start, end))
    x = torch.where(at5 < start5, kept, fresh) * (at5 < end5)
    x = x.view(B, H, 2, n // T, T, D)
    big = x.abs().amax((-1, -2), keepdim=True)
    scale = torch.where(big > 0, big / 127, torch.ones_like(big))
    x = ((x / scale).round().clamp(-127, 127) * scale).view(B, H, 2, n, D).to(tail.dtype)
    x = torch.where(at5 < end5, x, torch.zeros_like(x))
    # the newest block of each parity keeps its 16-bit rows
    last = (end - 1).clamp(min=0) // T                                               # (B, 1)
    blk = last - (last - torch.arange(2, device=DEV)) % 2                           # (B, 2): block kept in slot 0, 1
    pos = blk[:, :, None] * T + torch.arange(T, device=DEV)                         # (B, 2, T)
    put = (pos >= start[:, None]) & (pos < end[:, None])
    src = (st['cu'].long()[:-1, None, None] + pos - start[:, None]).clamp(0, new.shape[1] - 1)
    rows = new[:, src].permute(1, 4, 2, 0, 3, 5)                                     # (B, H, 2, 2, T, D)
    tail.copy_(torch.where(put[:, None, :, None, :, None], rows, tail))
    return dict(k=x[:, :, 0].transpose(1, 2).contiguous(), v=x[:, :, 1].transpose(1, 2).contiguous(), tail=tail)


def _rows(k8, v8):
    """Codes in the natural order, (B, H, tokens, D) each."""
    B, H, N, _, E = k8.shape[:5]
    k = k8.permute(0, 1, 2, 3, 5, 4, 6).reshape(B, H, N * T, E * 16)
    v = v8.view(B, H, N, E, 4, 16, 4, 4).permute(0, 1, 2, 6, 4, 7, 3, 5).reshape(B, H, N * T, E * 16)
    return k, v


def _attend(st):
    case = st['case']
    B, Hk, D, most = case['B'], case['Hk'], case['D'], st['most']
    G = case['Hq'] // Hk
    k, v = _rows(st['k8'], st['v8'])
    per = st['scale'].repeat_interleave(T, 2)
    k, v = k.float() * per[..., :1], v.float() * per[..., 1:]
    b, i = _owners(st)
    q = torch.zeros(B, most, case['Hq'], D, device=DEV)
    q[b, i] = st['q'].float()
    q = q.view(B, most, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, most * G, D)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(D)
    lens = st['lens'].long()
    count = st['cu'].long().diff()
    seen = lens[:, None] + (torch.arange(most, device=DEV) + 1 - count[:, None] if case['causal'] else torch.zeros(most, device=DEV).long())
    seen = torch.minimum(seen, lens[:, None]).repeat_interleave(G, 1)                # (B, most * G) keys a row sees
    s = s.masked_fill(torch.arange(k.shape[2], device=DEV) >= seen[:, None, :, None], float('-inf'))
    p = (s - s.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.view(B, Hk, most, G, D).permute(0, 2, 1, 3, 4).reshape(B, most, case['Hq'], D)
    return o[b, i].to(st['q'].dtype)


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    """Every input read once, every output written once. append: also the rows kept of the first block and the blocks read
    back; attend: the codes and scales of the cached rows."""
    size = dict(bf16=2, f16=2, f32=4)[case['dtype']]
    if case['kind'] == 'rope':
        M, R, heads = case['M'], case['R'], case['Hq'] + case['Hk']
        return dict(bytes=2 * M * heads * case['D'] * size + 4 * M * case['axes'] + 6 * R, flops=3 * M * heads * R)
    if case['kind'] == 'norm':
        M, K = case['M'], case['K']
        return dict(bytes=M * K * (3 * size + 1) + K * size + 4 * M, flops=8 * M * K)
    B, D = case['B'], case['D']
    start, new = _counts(case)
    if case['kind'] == 'append':
        rows = sum(new)
        touched = sum(s % T + n for s, n in zip(start, new))
        return dict(bytes=2 * case['H'] * D * (rows * size + (touched - rows) * size + touched + touched * size), flops=6 * touched * case['H'] * D)
    seen = sum(n * (s + n) - (n * (n - 1) // 2 if case['causal'] else 0) for s, n in zip(start, new))
    keys = sum(s + n for s, n in zip(start, new))
    return dict(bytes=2 * keys * case['Hk'] * D + keys * case['Hk'] // 8 + 2 * sum(new) * case['Hq'] * D * size, flops=4 * seen * case['Hq'] * D)


# ------------------------------------------------------------------------------------------ the same results in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case['kind'] == 'rope':
        h = case['R'] // 2
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), torch.stack([
            st['pos'][int(a)].double() * f for a, f in zip(st['axis'].tolist(), st['freq'].tolist())], 1) * (-1 if case['inverse'] else 1))
        out = {}
        for name in 'qk':
            x = st[name].double()
            z = torch.complex(x[..., :h], x[..., h:2 * h]) * turn[:, None]
            out[name] = torch.cat([z.real, z.imag, x[..., 2 * h:]], -1)
        return out
    if case['kind'] == 'norm':
        h = (st['x'].double() + st['r'].double()).to(st['x'].dtype).double()
        n = h / (h.pow(2).sum(1, keepdim=True) / case['K'] + 1e-6).sqrt() * (st['w'].double() + case['offset'])
        step = n.abs().max(1, keepdim=True).values / 127
        return dict(sum=h, scale=step[:, 0], values=torch.round(n / step) * step)
    start, lens, cu = (st[n].tolist() for n in ('start', 'lens', 'cu'))
    if case['kind'] == 'append':
        old, tail = st['tail'].double(), st['tail'].double()
        out = torch.zeros(2, case['B'], st['rows'], case['H'], case['D'], dtype=torch.float64, device=DEV)
        for b in range(case['B']):
            new = torch.stack([st['k'][cu[b]:cu[b + 1]], st['v'][cu[b]:cu[b + 1]]]).double()       # (2, m, H, D)
            j0 = start[b] // T
            kept = old[b, :, j0 % 2, :, :start[b] % T].permute(1, 2, 0, 3)
            rows = torch.cat([kept, new], 1)
            for j in range(0, rows.shape[1], T):
                part = rows[:, j:j + T]
                step = part.abs().amax((1, 3), keepdim=True) / 127
                out[:, b, j:j + part.shape[1]] = torch.round(part / step) * step
                if j + 2 * T >= rows.shape[1]:                                                     # one of the newest two blocks
                    lo = start[b] % T if j == 0 else 0
                    tail[b, :, (j0 + j // T) % 2, :, lo:part.shape[1]] = part[:, lo:].permute(2, 0, 1, 3)
        return dict(k=out[0], v=out[1], tail=tail)
    G = case['Hq'] // case['Hk']
    k, v = _rows(st['k8'], st['v8'])
    out = torch.zeros(st['q'].shape, dtype=torch.float64, device=DEV)
    for b in range(case['B']):
        m = cu[b + 1] - cu[b]
        for h in range(case['Hk']):
            step = st['scale'][b, h].double().repeat_interleave(T, 0)[:lens[b]]
            kd, vd = k[b, h, :lens[b]].double() * step[:, :1], v[b, h, :lens[b]].double() * step[:, 1:]
            for g in range(h * G, h * G + G):
                s = st['q'][cu[b]:cu[b + 1], g].double() @ kd.t() / case['D'] ** 0.5
                if case['causal']:
                    s += torch.full((m, lens[b]), -math.inf, dtype=torch.float64, device=DEV).triu(lens[b] - m + 1)
                out[cu[b]:cu[b + 1], g] = torch.softmax(s, 1) @ vd
    return out
