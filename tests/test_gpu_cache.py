"""Rotary positions, the paged cache and the attention over it against their definitions in 64 bits (oracle/cache_oracle.py).

Tolerances count roundings. A result rounded to its type is off by at most half a step, eps / 2 of its size (in fp16 by 2^-25 at
least). Rotary: a phase that is off by 2^-24 of half a turn, a sine and a cosine by 2 ulp, two products and a sum in 32 bits: under
6e-7 (|a| + |b|). Attention: a probability rounded to the type moves the output by eps / 2 of its share, together eps / 2 sum p |v|
(fp16: by 2^-25 of the largest probability each, at least); a score that is off by e moves it by 2 e sum p |v|, where D products
summed in 32 bits are off by at most D 2^-24 sum |q k|, and the base-2 exponent by a few 2^-24 of its size."""
import math
import threading

import pytest
import torch

import cache_oracle as O
import spargeattn_b200 as S
from spargeattn_b200 import ops

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _half_step(t, x):
    return torch.finfo(t).eps / 2 * x.abs() + {HF: 2.0 ** -25}.get(t, 0.0)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _status():
    """The device's word, cleared: 0 when nothing was reported since."""
    w = ops.device_status_word(torch.device("cuda", torch.cuda.current_device()))
    code = int(w.item())
    w.zero_()
    return code


@pytest.fixture(autouse=True)
def _nothing_reported():
    _status()
    yield
    torch.cuda.synchronize()
    assert _status() == 0


# ------------------------------------------------------------------------------------------------------------------ rotary
def _check_rotary(got, x, phase, interleaved, magnitude=1.0):
    want = O.rotary(x.cpu(), phase, interleaved, magnitude)
    room = _half_step(x.dtype, want) * 1.001 + 6e-7 * abs(magnitude) * O.rotary_size(x.cpu(), phase.shape[-1], interleaved)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert ((got.cpu().double() - want).abs() <= room).all()
    assert torch.equal(got.cpu()[..., 2 * phase.shape[-1]:], x.cpu()[..., 2 * phase.shape[-1]:])


# vectors of 8 and odd pair counts; one token, a block's border, several blocks
@pytest.mark.parametrize("D,pairs", [(128, 64), (128, 32), (64, 32), (64, 5), (80, 40), (6, 3), (256, 128), (30, 8)])
@pytest.mark.parametrize("dtype", [BF, HF, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_rotary(D, pairs, dtype, interleaved, layout):
    g = _gen(D + pairs)
    freq = S.rotary_frequencies(2 * pairs)[0]
    for B, N, Hq, Hk, far in ((1, 1, 3, 1, 1_000_003), (2, 9, 5, 2, 77), (1, 1300, 2, 2, 0)):
        shape = (lambda H: (B, H, N, D)) if layout == "HND" else (lambda H: (B, N, H, D))
        q, k = torch.randn(shape(Hq), generator=g).to(dtype), torch.randn(shape(Hk), generator=g).to(dtype)
        pos = far + torch.arange(N, dtype=torch.int32) + 1000 * torch.arange(B, dtype=torch.int32)[:, None]
        phase = (pos.double()[..., None] * freq.cpu()).unsqueeze(1 if layout == "HND" else 2)
        a, b = S.apply_rotary(q.cuda(), k.cuda(), pos.cuda(), freq, interleaved, magnitude=1.25, tensor_layout=layout)
        _check_rotary(a, q, phase, interleaved, 1.25)
        _check_rotary(b, k, phase, interleaved, 1.25)


def test_rotary_axes_views_and_empty():
    g = _gen(1)
    t, h, w, H, D = 3, 5, 7, 4, 128
    n = torch.arange(t * h * w)
    pos, sections = torch.stack([n // (h * w), n // w % h, n % w]), [22, 21, 21]
    freq = S.rotary_frequencies(D)[0]
    phase = torch.cat([pos[a].double()[:, None].expand(-1, s) for a, s in enumerate(sections)], -1) * freq.cpu()
    # q and k as slices of one projection, token-major, without a batch; int64 positions
    qkv = torch.randn(t * h * w, 3, H, D, generator=g).to(BF).cuda()
    q, k = qkv[:, 0], qkv[:, 1]
    for inter in (False, True):
        a, b = S.apply_rotary(q, k, pos.cuda(), freq, inter, sections, tensor_layout="NHD")
        _check_rotary(a, q, phase[:, None], inter)
        _check_rotary(b, k, phase[:, None], inter)
    # the same heads-first, seen through a transpose: the output keeps the storage order
    a = S.apply_rotary(q.transpose(0, 1), None, pos.cuda(), freq, True, sections)
    _check_rotary(a, q.transpose(0, 1), phase, True)
    # a batch in the positions' axes, an axis of no pairs, strided positions, rows that are not aligned, a last dimension that is not dense
    q = torch.randn(2, 2, 5, 65, generator=g).to(HF).cuda()[..., 1:]
    pos = torch.randint(0, 50, (2, 2, 10), generator=g).cuda()[:, :, ::2]
    a = S.apply_rotary(q, None, pos, freq[:32].contiguous(), False, [32, 0])
    _check_rotary(a, q, (pos[0].cpu().double()[..., None] * freq[:32].cpu())[:, None], False)
    q = torch.randn(1, 2, 64, 5, generator=g).cuda().transpose(2, 3)
    _check_rotary(S.apply_rotary(q, None, pos[0, :1], freq[:32].contiguous()), q, (pos[0, :1].cpu().double()[..., None] * freq[:32].cpu())[:, None], False)
    assert S.apply_rotary(q[:, :, :0], None, pos[0, :1, :0], freq[:32].contiguous()).shape == (1, 2, 0, 64)
    x = torch.tensor([math.inf, -math.inf, math.nan, 1.0] * 16, device="cuda", dtype=BF).view(1, 1, 1, 64)
    assert torch.equal(S.apply_rotary(x, None, pos[0, :1, :1], freq[:8].contiguous())[..., 16:].isnan(), x[..., 16:].isnan())


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(interleaved):
    g = _gen(2)
    freq = S.rotary_frequencies(48)[0]
    pos = torch.tensor([5, 90_000, 3], dtype=torch.int32)
    q, k = torch.randn(2, 3, 3, 64, generator=g), torch.randn(2, 1, 3, 64, generator=g)
    gq, gk = torch.randn(q.shape, generator=g), torch.randn(k.shape, generator=g)
    ql, kl = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    a, b = S.apply_rotary(ql, kl, pos.cuda(), freq, interleaved, magnitude=0.75)
    (a * gq.cuda()).sum().add((b * gk.cuda()).sum()).backward()
    phase = pos.double()[:, None] * freq.cpu()
    _check_rotary(ql.grad, gq, -phase, interleaved, 0.75)
    _check_rotary(kl.grad, gk, -phase, interleaved, 0.75)
    # by differences: a rotation is linear, so a step of any size gives the gradient along it
    d = torch.randn(q.shape, generator=g).cuda()
    f = lambda x: (S.apply_rotary(x, None, pos.cuda(), freq, interleaved, magnitude=0.75).double() * gq.cuda()).sum()  # noqa: E731
    diff, along = (f(q.cuda() + d) - f(q.cuda())).item(), (ql.grad.double() * d.double()).sum().item()
    # each of the 1152 values of two rotations, the step and the gradient is off by under 1e-6 of |x| + |y| <= 10
    assert abs(diff - along) <= 4 * 1152 * 1e-6 * 10
    # only one of them needs a gradient; a broadcast gradient; two backward passes
    a = S.apply_rotary(ql, k.cuda(), pos.cuda(), freq, interleaved)[0]
    one, = torch.autograd.grad(a.sum(), ql, retain_graph=True)
    _check_rotary(one, torch.ones_like(q), -phase, interleaved)
    assert torch.equal(torch.autograd.grad(a.sum(), ql)[0], one)
    b = S.apply_rotary(q.cuda(), kl, pos.cuda(), freq, interleaved)[1]
    _check_rotary(torch.autograd.grad(b.sum(), kl)[0], torch.ones_like(k), -phase, interleaved)
    # only one of the results is used
    a, b = S.apply_rotary(ql, kl, pos.cuda(), freq, interleaved)
    dq, dk = torch.autograd.grad(b.sum(), (ql, kl), allow_unused=True)
    assert dq is None
    _check_rotary(dk, torch.ones_like(k), -phase, interleaved)
    # the gradient of the gradient, in what it was taken along
    w = gq.cuda().requires_grad_()
    a = S.apply_rotary(ql, None, pos.cuda(), freq, interleaved)
    dq, = torch.autograd.grad(a, ql, w, create_graph=True)
    _check_rotary(torch.autograd.grad(dq, w, q.cuda())[0], q, phase, interleaved)
    with torch.no_grad():
        assert not S.apply_rotary(ql, None, pos.cuda(), freq, interleaved).requires_grad


# ------------------------------------------------------------------------------------------------------------------- cache
def _make(lengths, H, D, ps, dtype, seed, spare=3, dirt=math.nan, token_major=False):
    """Pages in random order; what lies behind the lengths, and in pages of nobody, is `dirt`."""
    g = _gen(seed)
    used = [-(-n // ps) for n in lengths]
    P, W = sum(used) + spare, max(used + [1]) + 1
    order = torch.randperm(P, generator=g).tolist()
    table = torch.full((len(lengths), W), -1, dtype=torch.int32)
    kp, vp = torch.full((P, H, ps, D), dirt, dtype=dtype), torch.full((P, H, ps, D), dirt, dtype=dtype)
    for i, n in enumerate(lengths):
        for e in range(used[i]):
            table[i, e] = page = order.pop()
            m = min(ps, n - e * ps)
            kp[page, :, :m] = torch.randn(H, m, D, generator=g).to(dtype)
            vp[page, :, :m] = torch.randn(H, m, D, generator=g).to(dtype)
    c = dict(k_pages=kp.cuda(), v_pages=vp.cuda(), page_table=table.cuda(), seq_lens=torch.tensor(lengths, dtype=torch.int32).cuda())
    if token_major:
        for n in ("k_pages", "v_pages"):
            c[n] = c[n].transpose(1, 2).contiguous().transpose(1, 2)
    return c


def _cu(chunks, start=0):
    return [start + sum(chunks[:i]) for i in range(len(chunks) + 1)]


def _check_attention(out, lse, q, c, lengths, cu, causal, scale=None):
    D = q.shape[-1]
    scale = D ** -0.5 if scale is None else scale
    table = [[p for p in r if p >= 0] for r in c["page_table"].tolist()]
    want, want_lse, weight, size = O.attention(q.cpu(), c["k_pages"].cpu(), c["v_pages"].cpu(), table, lengths, cu, causal, scale)
    e = (size * (D + 8) * 2.0 ** -24)[..., None]
    half = torch.finfo(q.dtype).eps / 2
    room = half * (want.abs() + weight) * 1.01 + 2 * e * weight + 1e-6 * weight
    if q.dtype == HF:   # small probabilities lose bits: 2^-25 of the largest each, against values of at most 6
        room = room + 2.0 ** -25 * (1 + 6 * max(lengths + [0]))
    rows = torch.zeros(q.shape[0], dtype=torch.bool)
    for a, b in zip(cu[:-1], cu[1:]):
        rows[a:b] = True
    off = ((out.cpu().double() - want).abs() - room)[rows]
    assert (off <= 0).all(), off.max()      # (a NaN is not)
    if lse is not None:
        got, none = lse.cpu().double()[rows], torch.isinf(want_lse[rows])
        assert torch.equal(got[none], want_lse[rows][none])
        assert ((got - want_lse[rows]).abs()[~none] <= (e[..., 0] + 2e-6 + 4e-7 * want_lse.abs())[rows][~none]).all()


SHAPES = [(1, 1), (4, 4), (8, 1), (6, 2), (20, 1), (16, 2), (40, 1)]


@pytest.mark.parametrize("Hq,Hkv", SHAPES)
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF), (64, BF), (128, HF)])
@pytest.mark.parametrize("ps", [16, 64, 256])
def test_decode(Hq, Hkv, D, dtype, ps):
    """One token per sequence: lengths of zero and one, at the borders of pages and tiles, long beside short."""
    lengths = [0, 1, 15, 16, 17, 127, 128, 129, 1000, 255, 2, 2900, 64]
    c = _make(lengths, Hkv, D, ps, dtype, Hq * D + ps)
    q = torch.randn(len(lengths), Hq, D, generator=_gen(3)).to(dtype).cuda()
    out, lse = S.paged_attention(q, **c, return_lse=True)
    _check_attention(out, lse, q, c, lengths, list(range(len(lengths) + 1)), True)
    assert torch.equal(out, S.paged_attention(q, **c, is_causal=False))          # one token sees all either way
    assert torch.equal(out, S.paged_attention(q, **c, cu_seqlens=torch.arange(len(lengths) + 1, dtype=torch.int32).cuda(), max_chunk=1))


@pytest.mark.parametrize("Hq,Hkv", SHAPES)
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF)])
@pytest.mark.parametrize("causal", [True, False])
def test_chunks(Hq, Hkv, D, dtype, causal):
    """Ragged chunks beside single tokens and sequences without any; lengths shorter than the chunk leave rows that see nothing."""
    chunks = [1, 0, 5, 130, 33, 300, 2, 70]
    lengths = [500, 77, 5, 131, 1000, 600, 1, 40]      # the last one: 30 rows before the first key
    for ps, token_major in ((32, False), (128, True)):
        c = _make(lengths, Hkv, D, ps, dtype, Hq + D, token_major=token_major)
        cu = _cu(chunks)
        q = torch.randn(cu[-1], Hq, D, generator=_gen(4)).to(dtype).cuda()
        cut = torch.tensor(cu, dtype=torch.int32).cuda()
        out, lse = S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=300, is_causal=causal, return_lse=True)
        _check_attention(out, lse, q, c, lengths, cu, causal)
        # a bound that is too small, or none, may choose another kernel: results hold
        for most in (None, 1):
            o2, l2 = S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=most, is_causal=causal, return_lse=True)
            _check_attention(o2, l2, q, c, lengths, cu, causal)


# more sequences than threads of a CTA; some hold nothing, some bring nothing; one long one among them
@pytest.mark.parametrize("sequences,most", [(700, 1), (700, 3), (1500, 40)])
def test_many_sequences(sequences, most):
    g = _gen(sequences + most)
    H, D, ps = 2, 64, 16
    chunks = [1] * sequences if most == 1 else torch.randint(0, most + 1, (sequences,), generator=g).tolist()
    lengths = torch.randint(0, 90, (sequences,), generator=g).tolist()
    lengths[sequences // 3] = 3000
    c = _make(lengths, H, D, ps, HF, sequences)
    cu = _cu(chunks)
    q = torch.randn(cu[-1], 3 * H, D, generator=g).to(HF).cuda()
    cut = None if most == 1 else torch.tensor(cu, dtype=torch.int32).cuda()
    out, lse = S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=most, return_lse=True)
    _check_attention(out, lse, q, c, lengths, cu, True)


@pytest.mark.parametrize("ps", [16, 256])
@pytest.mark.parametrize("D,dtype", [(128, HF), (64, BF)])
@pytest.mark.parametrize("Hq,Hkv", [(66, 33), (128, 1)])
def test_chunks_of_many_heads(ps, D, dtype, Hq, Hkv):
    chunks, lengths = [3, 17], [300, 1025]
    c = _make(lengths, Hkv, D, ps, dtype, Hq + ps)
    q = torch.randn(20, Hq, D, generator=_gen(19)).to(dtype).cuda()
    for causal in (True, False):
        out, lse = S.paged_attention(q, **c, cu_seqlens=torch.tensor([0, 3, 20], dtype=torch.int32).cuda(), max_chunk=17, is_causal=causal, return_lse=True)
        _check_attention(out, lse, q, c, lengths, [0, 3, 20], causal)


def test_dimensions_of_one_have_no_stride():
    """What a view says about a dimension of size one is not looked at."""
    c = _make([100], 1, 64, 16, BF, 22, spare=0)
    q = torch.randn(1, 4, 64, generator=_gen(22)).to(BF).cuda()
    want = S.paged_attention(q, **c)
    P = c["k_pages"].shape[0]
    for n in ("k_pages", "v_pages"):
        c[n] = c[n].as_strided((P, 1, 16, 64), (16 * 64, 3, 64, 1))
    out = torch.zeros(300, dtype=BF, device="cuda")[:256].as_strided((1, 4, 64), (5, 64, 1))
    assert torch.equal(S.paged_attention(q.as_strided((1, 4, 64), (7, 64, 1)), **c, out=out), want)
    k = torch.randn(1, 1, 64, generator=_gen(23)).to(BF).cuda()
    S.append_kv(k.as_strided((1, 1, 64), (1, 1, 1)), k, **c)
    assert torch.equal(c["k_pages"][c["page_table"][0, 6], :, 3], k[0])


def test_output_over_the_queries():
    """Every row of q is read before its output is written: out may be q itself."""
    for chunk, length in ((1, 5000), (300, 2000)):
        c = _make([length, 77], 1, 64, 16, BF, chunk)
        q = torch.randn(2 * chunk, 4, 64, generator=_gen(20)).to(BF).cuda()
        cut = torch.tensor([0, chunk, 2 * chunk], dtype=torch.int32).cuda()
        want = S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=chunk)
        assert torch.equal(S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=chunk, out=q), want) and torch.equal(q, want)


@pytest.mark.parametrize("Hq,Hkv,chunk,length", [(8, 2, 3, 9001), (4, 1, 64, 20_000), (32, 4, 500, 2500), (2, 2, 1, 40_000)])
def test_long_axis(Hq, Hkv, chunk, length):
    """Few rows over a long axis: many CTAs work on one tile and their parts are joined."""
    for D, dtype in ((128, BF), (64, HF)):
        c = _make([length, 7], Hkv, D, 64, dtype, length)
        cu = [0, chunk, chunk + 1]
        q = (2 * torch.randn(chunk + 1, Hq, D, generator=_gen(5))).to(dtype).cuda()
        out, lse = S.paged_attention(q, **c, cu_seqlens=torch.tensor(cu, dtype=torch.int32).cuda(), max_chunk=chunk, return_lse=True)
        _check_attention(out, lse, q, c, [length, 7], cu, True)
        again = S.paged_attention(q, **c, cu_seqlens=torch.tensor(cu, dtype=torch.int32).cuda(), max_chunk=chunk)
        assert torch.equal(out, again)


@pytest.mark.parametrize("chunk", [1, 200])
def test_rows_of_no_sequence_and_given_out(chunk):
    H, D = 4, 64
    lengths, chunks = [300, 250], [chunk, chunk]
    c = _make(lengths, 2, D, 16, BF, 6)
    cu = _cu(chunks, start=3)
    T = cu[-1] + 5
    # q and out as slices of wider tensors
    q = torch.randn(T, H + 2, D, generator=_gen(6)).to(BF).cuda()[:, 1:-1]
    wide = torch.full((T, H, 2 * D), 7.0, dtype=BF, device="cuda")
    cut = torch.tensor(cu, dtype=torch.int32).cuda()
    out = wide[:, :, D:]
    assert S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=chunk, out=out).data_ptr() == out.data_ptr()
    _check_attention(out, None, q, c, lengths, cu, True)
    assert (wide[:, :, :D] == 7).all() and (out[:3] == 7).all() and (out[cu[-1]:] == 7).all()
    fresh, lse = S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=chunk, return_lse=True)
    assert torch.equal(fresh[3: cu[-1]], out[3: cu[-1]])
    for t in (fresh[:3], fresh[cu[-1]:]):
        assert (t == 0).all()
    assert (lse[:3] == -math.inf).all() and (lse[cu[-1]:] == -math.inf).all()
    # nothing at all
    none = torch.zeros(3, dtype=torch.int32).cuda()
    assert (S.paged_attention(q, **c, cu_seqlens=none) == 0).all()
    assert S.paged_attention(q[:0], **c, cu_seqlens=none).shape == (0, H, D)
    # cu_seqlens that run backwards or past the tokens reach no other memory
    odd = torch.tensor([2, T + 50, 1], dtype=torch.int32).cuda()
    assert S.paged_attention(q, **c, cu_seqlens=odd, max_chunk=chunk).shape == q.shape


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
@pytest.mark.parametrize("chunk", [1, 150])
def test_scales_and_extreme_scores(scale, chunk):
    H, D = 2, 64
    c = _make([400], H, D, 16, BF, 7)
    q = torch.randn(chunk, H, D, generator=_gen(7)).to(BF).cuda()
    cut = torch.tensor([0, chunk], dtype=torch.int32).cuda()
    out, lse = S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=chunk, scale=scale, return_lse=True)
    _check_attention(out, lse, q, c, [400], [0, chunk], True, scale)
    # keys of the type's lowest value: scores near -10^38 are scores, and softmax over equal ones is a mean
    low = dict(c, k_pages=torch.full_like(c["k_pages"], torch.finfo(BF).min / 128))
    ones = torch.ones_like(q)
    out = S.paged_attention(ones, **low, cu_seqlens=cut, max_chunk=chunk, is_causal=False, scale=1.0)
    pages = c["page_table"][0, :25].long()
    mean = c["v_pages"][pages].transpose(0, 1).reshape(H, -1, D)[:, :400].double().mean(1)
    assert (out.double() - mean).abs().max() <= 2 * 2.0 ** -8 * c["v_pages"][pages].transpose(0, 1).reshape(H, -1, D)[:, :400].float().abs().max()


@pytest.mark.parametrize("chunk", [1, 150])
def test_a_row_that_is_not_a_number_stays_one(chunk):
    c = _make([300], 1, 64, 32, BF, 7)
    q = torch.randn(chunk, 2, 64, generator=_gen(7)).to(BF).cuda()
    cut = torch.tensor([0, chunk], dtype=torch.int32).cuda()
    good = S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=chunk)
    q[chunk // 2, 1, 3] = math.nan
    out, lse = S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=chunk, return_lse=True)
    assert out[chunk // 2, 1].isnan().all() and lse[chunk // 2, 1].isnan()
    good[chunk // 2, 1] = out[chunk // 2, 1] = 0
    assert torch.equal(out, good)


@pytest.mark.parametrize("chunk", [1, 40])
def test_bad_pages_are_reported_and_harmless(chunk):
    H, D = 2, 64
    lengths = [100, 90]
    c = _make(lengths, H, D, 16, BF, 8)
    q = torch.randn(2 * chunk, H, D, generator=_gen(8)).to(BF).cuda()
    cut = torch.tensor([0, chunk, 2 * chunk], dtype=torch.int32).cuda()
    good = S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=chunk)
    assert _status() == 0
    for bad in (-1, c["k_pages"].shape[0], 2 ** 31 - 1, -2 ** 31):
        table = c["page_table"].clone()
        table[0, 2] = bad
        out = S.paged_attention(q, **dict(c, page_table=table), cu_seqlens=cut, max_chunk=chunk)
        with pytest.raises(RuntimeError, match="does not have"):
            ops.check_device_status()
        assert _status() == 4 and torch.equal(out[chunk:], good[chunk:])
    for bad in (-5, 2 ** 31 - 1):
        lens = c["seq_lens"].clone()
        lens[0] = bad
        out = S.paged_attention(q, **dict(c, seq_lens=lens), cu_seqlens=cut, max_chunk=chunk)
        assert _status() == 4 and torch.equal(out[chunk:], good[chunk:])


def test_pages_far_into_a_large_pool():
    """Offsets that pass 32 bits, in elements and in bytes."""
    H, D, ps = 8, 128, 64
    P = (2 ** 31) // (H * ps * D) + 8            # 2^31 elements and some
    kp, vp = (torch.zeros(P, H, ps, D, dtype=BF, device="cuda") for _ in range(2))
    g = _gen(9)
    lengths, used = [150, 70], [3, 2]
    table = torch.full((2, 4), -1, dtype=torch.int32)
    table[0, :3], table[1, :2] = torch.tensor([P - 1, 0, P - 3]), torch.tensor([P - 2, P - 4])
    c = dict(k_pages=kp, v_pages=vp, page_table=table.cuda(), seq_lens=torch.tensor(lengths, dtype=torch.int32).cuda())
    k, v = (torch.randn(220, H, D, generator=g).to(BF).cuda() for _ in range(2))
    cu = [0, 150, 220]
    cut = torch.tensor(cu, dtype=torch.int32).cuda()
    S.append_kv(k, v, **c, cu_seqlens=cut)
    for i in range(2):
        pages = table[i, : used[i]].long().cuda()
        assert torch.equal(kp[pages].transpose(0, 1).reshape(H, -1, D)[:, : lengths[i]].transpose(0, 1), k[cu[i]: cu[i + 1]])
        assert torch.equal(vp[pages].transpose(0, 1).reshape(H, -1, D)[:, : lengths[i]].transpose(0, 1), v[cu[i]: cu[i + 1]])
    small, rename = [P - 1, 0, P - 3, P - 2, P - 4], {}
    rename = {p: i for i, p in enumerate(small)}
    c2 = dict(k_pages=kp[small], v_pages=vp[small], seq_lens=c["seq_lens"],
              page_table=torch.tensor([[rename.get(p, -1) for p in r] for r in table.tolist()], dtype=torch.int32).cuda())
    q = torch.randn(220, 2 * H, D, generator=g).to(BF).cuda()
    assert torch.equal(S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=150), S.paged_attention(q, **c2, cu_seqlens=cut, max_chunk=150))
    one = S.paged_attention(q[:2], **c)
    assert torch.equal(one, S.paged_attention(q[:2], **c2))


# ------------------------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("D,dtype,ps", [(64, BF, 16), (128, HF, 64), (80, BF, 32)])
@pytest.mark.parametrize("how", ["plain", "half", "interleaved", "partial"])
def test_append(D, dtype, ps, how):
    H, Hq = 2, 6
    chunks, lengths = [1, 0, 40, 17, 1], [1, 5, 133, 17, 1000]
    c = _make(lengths, H, D, ps, dtype, D + ps, dirt=3.0)
    before_k, before_v = c["k_pages"].cpu(), c["v_pages"].cpu()
    cu = _cu(chunks, start=2)
    T = cu[-1] + 3
    g = _gen(10)
    qkv = torch.randn(T, Hq + 2 * H, D, generator=g).to(dtype).cuda()
    q, k, v = qkv[:, :Hq], qkv[:, Hq: Hq + H], qkv[:, Hq + H:]
    freq = None if how == "plain" else S.rotary_frequencies(D // 2 if how == "partial" else D)[0]
    inter = how == "interleaved"
    got = S.append_kv(k, v, **c, cu_seqlens=torch.tensor(cu, dtype=torch.int32).cuda(), q=None if how == "plain" else q, frequencies=freq,
                      interleaved=inter, magnitude=1.0 if how == "plain" else 1.5)
    where = O.rows(lengths, cu)
    want_k, want_v = before_k.clone(), before_v.clone()
    table = c["page_table"].tolist()
    for t in range(T):
        if t not in where:
            assert how == "plain" or (got[t] == 0).all()
            continue
        i, p = where[t]
        page, at = table[i][p // ps], p % ps
        want_v[page, :, at] = v[t].cpu()
        if how == "plain":
            want_k[page, :, at] = k[t].cpu()
        else:
            phase = p * freq.cpu()
            _check_rotary(c["k_pages"][page, :, at], k[t], phase, inter, 1.5)
            _check_rotary(got[t], q[t], phase, inter, 1.5)
            want_k[page, :, at] = c["k_pages"][page, :, at].cpu()
    assert got is None if how == "plain" else got.shape == q.shape
    assert torch.equal(c["v_pages"].cpu(), want_v) and torch.equal(c["k_pages"].cpu(), want_k)      # nothing else was written


def test_append_leaves_out_what_has_no_page():
    H, D = 2, 64
    c = _make([20, 40, 10], H, D, 16, BF, 11, dirt=3.0)
    k = torch.randn(3, H, D, generator=_gen(11)).to(BF).cuda()
    before = c["k_pages"].clone()
    table, lens = c["page_table"].clone(), c["seq_lens"].clone()
    table[0, 1] = 2 ** 30
    table[1, 2] = -7
    lens[2] = 0                                                        # a token in front of the first position
    S.append_kv(k, k, c["k_pages"], c["v_pages"], table, lens)
    assert _status() == 4 and torch.equal(c["k_pages"], before)
    lens[:] = 2 ** 31 - 1
    S.append_kv(k, k, c["k_pages"], c["v_pages"], table, lens)
    assert _status() == 4 and torch.equal(c["k_pages"], before)


# ------------------------------------------------------------------------------------------------------------- bookkeeping
def _pool(P, ps, sequences, width, seed, slices=(3, 2), H=2, D=64):
    """A pool in use, the oracle's copy of it, and the pages left over."""
    g = _gen(seed)
    pages = torch.randn(*slices, P, H, ps, D, generator=g).to(BF)
    lens = torch.randint(0, (width - 2) * ps, (sequences,), generator=g).tolist()
    lens[0], lens[1] = 0, 2 * ps                                       # an empty one, one that ends with a page
    order = torch.randperm(P, generator=g).tolist()
    table, refs = [[-1] * width for _ in lens], [0] * P
    for i, n in enumerate(lens):
        for e in range(-(-n // ps)):
            table[i][e] = order.pop()
            refs[table[i][e]] = 1
    o = O.Pool(table, lens, refs, pages.flatten(0, len(slices) - 1).clone(), ps)
    dev = [torch.tensor(x, dtype=torch.int32).cuda() for x in (table, lens, refs)]
    return pages.cuda(), *dev, o


def _same(pages, table, lens, refs, o):
    assert table.tolist() == o.table and lens.tolist() == o.lens and refs.tolist() == o.refs
    n = pages.dim() - 4
    assert torch.equal(pages.cpu().flatten(0, n - 1) if n else pages.cpu()[None], o.pages)


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32).cuda()


# more sequences than the plan's threads; a pool of several rounds of 8 192 pages; one that is not a multiple of anything
@pytest.mark.parametrize("P,sequences,width", [(64, 5, 6), (1999, 37, 12), (20_003, 1500, 9)])
def test_allocate_fork_free_compact(P, sequences, width):
    ps = 16
    slices, H, D = ((3, 2), 2, 64) if P < 10_000 else ((1,), 1, 64)
    pages, table, lens, refs, o = _pool(P, ps, sequences, width, P, slices, H, D)
    g = _gen(12)
    _same(pages, table, lens, refs, o)
    for step in range(4):
        new = torch.randint(0, 2 * ps, (sequences,), generator=g).tolist()
        new[step] = -3 if step == 1 else 10 ** 9 if step == 2 else 0
        served = S.allocate_pages(table, lens, refs, _i32(*new), ps)
        assert served.tolist() == o.allocate(new)
        n = sequences // 2
        src, dst = torch.randint(0, sequences, (n,), generator=g).tolist(), torch.randperm(sequences, generator=g)[:n].tolist()
        if n > 1:
            dst[0] = dst[-1]                                           # the same destination twice: the later pair has it
            src[1] = dst[1]                                            # its own source
        assert S.fork_sequences(pages, table, lens, refs, _i32(*src), _i32(*dst)).tolist() == o.fork(src, dst)
        _same(pages, table, lens, refs, o)
        gone = torch.randperm(sequences, generator=g)[: sequences // 3].tolist() + [-1]
        S.free_sequences(table, lens, refs, _i32(*gone, *gone), ps)    # twice each
        o.free(gone)
        if step == 2:
            assert S.compact_pages(pages, table, refs).tolist() == [o.compact()]
        _same(pages, table, lens, refs, o)
    assert S.compact_pages(pages, table, refs).tolist() == [o.compact()]
    _same(pages, table, lens, refs, o)
    assert S.compact_pages(pages, table, refs).item() == sum(r > 0 for r in o.refs)      # nothing left to move
    _same(pages, table, lens, refs, o)


def test_pool_runs_out():
    ps = 16
    table, lens, refs = torch.full((4, 3), -1, dtype=torch.int32).cuda(), _i32(0, 0, 0, 0), torch.zeros(5, dtype=torch.int32).cuda()
    assert S.allocate_pages(table, lens, refs, _i32(33, 20, 1, 0), ps).tolist() == [True, True, False, True]
    assert table.tolist() == [[0, 1, 2], [3, 4, -1], [-1, -1, -1], [-1, -1, -1]] and lens.tolist() == [33, 20, 0, 0]
    assert S.allocate_pages(table, lens, refs, _i32(15, 12, 1, 0), ps).tolist() == [True, True, False, True]     # within their pages
    pages = torch.randn(5, 1, ps, 64).to(BF).cuda()
    assert S.allocate_pages(table, lens, refs, _i32(0, -1, 0, 0), ps).tolist() == [True, False, True, True]
    S.free_sequences(table, lens, refs, _i32(0))
    assert S.allocate_pages(table, lens, refs, _i32(0, 0, 18, 17), ps).tolist() == [True, True, True, False]
    assert table.tolist()[2] == [0, 1, -1] and refs.tolist() == [1, 1, 0, 1, 1]
    # two forks of a sequence with a part of a page, room for one
    assert S.fork_sequences(pages, table, lens, refs, _i32(2, 2), _i32(0, 3)).tolist() == [True, False]
    assert table.tolist()[0] == [0, 2, -1] and refs.tolist() == [2, 1, 1, 1, 1] and torch.equal(pages[2], pages[1])
    # numbers of sequences that there are not
    assert S.fork_sequences(pages, table, lens, refs, _i32(7, -1, 0), _i32(3, 3, -1)).tolist() == [False, False, False]
    assert _status() == 4
    S.free_sequences(table, lens, refs, _i32(4))
    assert _status() == 4
    # nothing to do, and no pool
    empty = _i32()
    S.free_sequences(table, lens, refs, empty)
    assert S.fork_sequences(pages, table, lens, refs, empty, empty).shape == (0,)
    assert S.allocate_pages(table[:0], lens[:0], refs, empty, ps).shape == (0,)


def test_captured_bookkeeping():
    """Forks, growth, release and compaction in one graph, replayed over a pool that goes on changing."""
    ps = 16
    pages, table, lens, refs, o = _pool(300, ps, 12, 10, 21)
    src, dst, new, gone = _i32(2, 3, 4), _i32(5, 6, 2), torch.full((12,), 3, dtype=torch.int32).cuda(), _i32(7, -1)
    ops.device_status_word(pages.device)

    def step():
        S.fork_sequences(pages, table, lens, refs, src, dst)
        served = S.allocate_pages(table, lens, refs, new, ps)
        S.free_sequences(table, lens, refs, gone)
        return served, S.compact_pages(pages, table, refs)

    def want():
        o.fork(src.tolist(), dst.tolist())
        served = o.allocate(new.tolist())
        o.free(gone.tolist())
        return served, [o.compact()]

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        served, live = step()
    for n in range(4):
        graph.replay()
        assert (served.tolist(), live.tolist()) == want()
        _same(pages, table, lens, refs, o)
        src.copy_(_i32(n, 8, 9)), dst.copy_(_i32(11, n + 1, 10)), gone.copy_(_i32(n + 4, n + 4))


def test_copy_pages():
    g = _gen(13)
    for shape in ((2, 3, 9, 2, 16, 64), (40, 1, 16, 8), (3, 5, 4, 32, 128)):
        pages = torch.randn(shape, generator=g).to(BF)
        want, dev = pages.clone(), pages.cuda()
        src, dst = [0, 1, 0, -1], [3, 4, 2, 0]
        S.copy_pages(dev, _i32(*src), _i32(*dst))
        for a, b in zip(src, dst):
            if a >= 0:
                want.select(-4, b).copy_(pages.select(-4, a))
        assert torch.equal(dev.cpu(), want)
    # layers apart: a view of every other slice; a page onto itself
    dev = torch.randn(6, 9, 1, 16, 8, generator=g).cuda()
    before = dev.clone()
    S.copy_pages(dev[::2], _i32(5, 7), _i32(6, 7))
    before[::2, 6] = before[::2, 5]
    assert torch.equal(dev, before)
    S.copy_pages(dev, _i32(), _i32())
    # a destination twice, or one that is a source: not copied, the others are
    S.copy_pages(dev, _i32(0, 1, 2), _i32(3, 3, 4))
    assert _status() == 5
    before[:, 4] = before[:, 2]
    assert torch.equal(dev, before)
    S.copy_pages(dev, _i32(0, 1), _i32(1, 2))
    assert _status() == 5
    before[:, 2] = before[:, 1]
    assert torch.equal(dev, before)
    S.copy_pages(dev, _i32(0, 9), _i32(9, 0))
    assert _status() == 4 and torch.equal(dev, before)


# ---------------------------------------------------------------------------------------------------------------- together
class _Conversations:
    """A two-layer cache and what it should hold, kept as whole tensors per sequence."""

    def __init__(self, sequences, Hq, Hkv, D, ps, dtype, P, width):
        self.Hq, self.Hkv, self.D, self.ps, self.dtype = Hq, Hkv, D, ps, dtype
        self.pages = torch.full((2, 2, P, Hkv, ps, D), math.nan, dtype=dtype, device="cuda")
        self.table = torch.full((sequences, width), -1, dtype=torch.int32).cuda()
        self.lens, self.refs = torch.zeros(sequences, dtype=torch.int32).cuda(), torch.zeros(P, dtype=torch.int32).cuda()
        self.freq = S.rotary_frequencies(D)[0]
        self.held = [[torch.zeros(2, 0, Hkv, D, dtype=dtype) for _ in range(sequences)] for _ in range(2)]

    def step(self, chunks, g):
        assert S.allocate_pages(self.table, self.lens, self.refs, _i32(*chunks), self.ps).all()
        cu, T = _cu(chunks), sum(chunks)
        cut = torch.tensor(cu, dtype=torch.int32).cuda()
        for layer in range(2):
            q, k, v = (torch.randn(T, h, self.D, generator=g).to(self.dtype) for h in (self.Hq, self.Hkv, self.Hkv))
            kp, vp = self.pages[layer, 0], self.pages[layer, 1]
            turned = S.append_kv(k.cuda(), v.cuda(), kp, vp, self.table, self.lens, cut, q=q.cuda(), frequencies=self.freq)
            out = S.paged_attention(turned, kp, vp, self.table, self.lens, cut, max_chunk=max(chunks))
            lengths = self.lens.tolist()
            for i in range(len(chunks)):
                at = torch.arange(lengths[i] - chunks[i], lengths[i], dtype=torch.int32)
                kt = S.apply_rotary(k[cu[i]: cu[i + 1]].cuda(), None, at.cuda(), self.freq, tensor_layout="NHD").cpu()
                self.held[layer][i] = torch.cat([self.held[layer][i], torch.stack([kt, v[cu[i]: cu[i + 1]]])], 1)
                assert self.held[layer][i].shape[1] == lengths[i]
            # the same sequences as a cache of one page each: what was held, not what the pages say
            for i in range(len(chunks)):
                if chunks[i] == 0:
                    continue
                h = self.held[layer][i]
                c = dict(k_pages=h[0].transpose(0, 1)[None], v_pages=h[1].transpose(0, 1)[None], page_table=torch.zeros(1, 1, dtype=torch.int32))
                rows = slice(cu[i], cu[i + 1])
                _check_attention(out[rows], None, turned[rows], c, [lengths[i]], [0, chunks[i]], True)

    def fork(self, src, dst):
        assert S.fork_sequences(self.pages, self.table, self.lens, self.refs, _i32(*src), _i32(*dst)).all()
        for layer in self.held:
            new = {d: layer[s].clone() for s, d in zip(src, dst)}
            for d, h in new.items():
                layer[d] = h

    def free(self, which):
        S.free_sequences(self.table, self.lens, self.refs, _i32(*which))
        for layer in self.held:
            for i in which:
                layer[i] = layer[i][:, :0]


@pytest.mark.parametrize("D,dtype,Hq,Hkv,ps", [(64, BF, 4, 2, 16), (128, HF, 6, 1, 32)])
def test_conversations(D, dtype, Hq, Hkv, ps):
    g = _gen(14)
    t = _Conversations(4, Hq, Hkv, D, ps, dtype, 120, 30)
    t.step([37, 5, 200, 0], g)                     # prompts
    t.step([1, 1, 1, 1], g)
    t.fork([2, 0], [3, 1])                         # two of them go on twice
    t.step([1, 1, 1, 1], g)                        # forks write behind the same past, each in its own page
    t.step([1, 3, 0, 90], g)
    t.fork([1, 2, 3, 0], [0, 1, 2, 3])             # beams in another order
    t.step([1, 1, 1, 1], g)
    t.free([0, 2])
    assert S.compact_pages(t.pages, t.table, t.refs).item() == int((t.refs > 0).sum())
    t.step([20, 1, 64, 1], g)
    t.free([0, 1, 2, 3])
    assert not t.refs.any() and (t.table == -1).all()


def test_captured_step_follows_lengths():
    """A captured step is replayed over growing lengths, tables that change and another split of the tokens."""
    g = _gen(15)
    B, Hq, Hkv, D, ps, P = 3, 8, 2, 64, 16, 200
    kv = torch.full((2, P, Hkv, ps, D), math.nan, dtype=BF, device="cuda")
    table, lens, refs = torch.full((B, 60), -1, dtype=torch.int32).cuda(), _i32(0, 0, 0), torch.zeros(P, dtype=torch.int32).cuda()
    freq = S.rotary_frequencies(D)[0]
    T = 24
    new, cut = _i32(0, 0, 0), _i32(0, 0, 0, 0)
    q, k, v = (torch.zeros(T, h, D, dtype=BF, device="cuda") for h in (Hq, Hkv, Hkv))
    ops.device_status_word(q.device)

    def step():
        S.allocate_pages(table, lens, refs, new, ps)
        turned = S.append_kv(k, v, kv[0], kv[1], table, lens, cut, q=q, frequencies=freq)
        return turned, *S.paged_attention(turned, kv[0], kv[1], table, lens, cut, max_chunk=T, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):          # two graphs of the same step: their workspaces are their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    for n, chunks in enumerate([[24, 0, 0], [1, 20, 3], [8, 8, 8], [1, 1, 1], [0, 0, 24]]):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g))
        new.copy_(_i32(*chunks))
        cut.copy_(_i32(*_cu(chunks)))
        graph, (turned, out, lse) = graphs[n % 2]
        graph.replay()
        c = dict(k_pages=kv[0], v_pages=kv[1], page_table=table)
        _check_attention(out, lse, turned, c, lens.tolist(), _cu(chunks), True)
        assert (out[sum(chunks):] == 0).all()


def test_rotary_backward_captured():
    """A training step of its own graph, and an eager one of the same leaves afterwards."""
    freq = S.rotary_frequencies(64)[0]
    pos = torch.arange(70, dtype=torch.int32).cuda()
    q = torch.randn(1, 2, 70, 64, generator=_gen(16)).cuda().requires_grad_()
    gq = torch.randn(1, 2, 70, 64, generator=_gen(17)).cuda()

    def step():
        return torch.autograd.grad(S.apply_rotary(q, None, pos, freq), q, gq)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dq = step()
    graph.replay()
    assert torch.equal(dq, step())


def test_streams_and_threads():
    """Calls on several threads and streams at once: each has its own workspace."""
    g = _gen(18)
    work = []
    for i, (lengths, Hq, Hkv, D, chunk) in enumerate([([5000, 31], 8, 1, 128, 1), ([900, 900, 30], 4, 4, 64, 1), ([700, 2600], 16, 2, 64, 300)]):
        c = _make(lengths, Hkv, D, 32, BF, 100 + i)
        q = torch.randn(len(lengths) * chunk, Hq, D, generator=g).to(BF).cuda()
        cut = torch.tensor(_cu([chunk] * len(lengths)), dtype=torch.int32).cuda()
        work.append((c, q, cut, chunk, lengths, S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=chunk)))
    torch.cuda.synchronize()
    wrong = []

    def run(c, q, cut, chunk, lengths, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not torch.equal(S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=chunk), want):
                    wrong.append(lengths)

    threads = [threading.Thread(target=run, args=w) for w in work for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("chunk", [1, 200])
def test_lse_of_rows_of_no_sequence_beside_a_given_out(chunk):
    """The lse is the call's own tensor: rows of no sequence are -inf there, also where a given out keeps what it had."""
    H, D = 4, 64
    lengths, chunks = [300, 250], [chunk, chunk]
    c = _make(lengths, 2, D, 16, BF, 24)
    cu = _cu(chunks, start=3)
    T = cu[-1] + 5
    q = torch.randn(T, H, D, generator=_gen(24)).to(BF).cuda()
    cut = torch.tensor(cu, dtype=torch.int32).cuda()
    want, want_lse = S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=chunk, return_lse=True)
    out = torch.full_like(q, 7.0)
    stale = torch.full((T, H), 7.0, device="cuda")                     # what the call's own tensor may find in its memory
    del stale
    _, lse = S.paged_attention(q, **c, cu_seqlens=cut, max_chunk=chunk, out=out, return_lse=True)
    assert torch.equal(lse, want_lse) and (lse[:3] == -math.inf).all() and (lse[cu[-1]:] == -math.inf).all()
    assert torch.equal(out[3: cu[-1]], want[3: cu[-1]]) and (out[:3] == 7).all() and (out[cu[-1]:] == 7).all()
    # no sequence at all
    none = dict(c, page_table=c["page_table"][:0], seq_lens=c["seq_lens"][:0], cu_seqlens=_i32(0), max_chunk=chunk)
    out, lse = S.paged_attention(q, **none, out=torch.full_like(q, 7.0), return_lse=True)
    assert (out == 7).all() and (lse == -math.inf).all()
    out, lse = S.paged_attention(q, **none, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("H", [1, 2, 16])
def test_bookkeeping_of_token_major_pages(H):
    """Pages [page_size, kv_heads, D] seen through a transpose, as append_kv and paged_attention take them."""
    ps = 32
    pages, table, lens, refs, o = _pool(150, ps, 9, 7, H, H=H)
    if H == 1:                                                         # what a view says about one head is not looked at
        pages = pages.as_strided(pages.shape, (*pages.stride()[:-3], 3, *pages.stride()[-2:]))
    else:
        pages = pages.transpose(-2, -3).contiguous().transpose(-2, -3)
        assert pages.stride(-3) == 64
    g = _gen(25)
    for step in range(3):
        src, dst = torch.randint(0, 9, (4,), generator=g).tolist(), torch.randperm(9, generator=g)[:4].tolist()
        assert S.fork_sequences(pages, table, lens, refs, _i32(*src), _i32(*dst)).tolist() == o.fork(src, dst)
        new = torch.randint(0, ps, (9,), generator=g).tolist()
        assert S.allocate_pages(table, lens, refs, _i32(*new), ps).tolist() == o.allocate(new)
        gone = [step, 5 + step]
        S.free_sequences(table, lens, refs, _i32(*gone))
        o.free(gone)
        _same(pages, table, lens, refs, o)
        assert S.compact_pages(pages, table, refs).tolist() == [o.compact()]
        _same(pages, table, lens, refs, o)
    S.copy_pages(pages, _i32(140, 3), _i32(149, 148))
    o.pages[:, 149], o.pages[:, 148] = o.pages[:, 140], o.pages[:, 3]
    _same(pages, table, lens, refs, o)


def test_skipped_copies_stand_in_no_ones_way():
    """A pair that is skipped, for a -1 or a page that the pool does not have, takes no part in the search for hazards."""
    dev = torch.randn(2, 9, 1, 16, 8, generator=_gen(26)).cuda()
    want = dev.clone()
    # 0 -> 3 beside pairs that name page 3, or page 0, and copy nothing
    S.copy_pages(dev, _i32(0, -1, 3, -1, 5), _i32(3, 3, -1, 0, 6))
    want[:, 3], want[:, 6] = want[:, 0], want[:, 5]
    assert _status() == 0 and torch.equal(dev, want)
    S.copy_pages(dev, _i32(1, 9, 4, -5), _i32(4, 4, 2 ** 30, 1))
    want[:, 4] = want[:, 1]
    assert _status() == 4 and torch.equal(dev, want)


# few pairs, planned in one kernel, and many
@pytest.mark.parametrize("n", [3, 600])
def test_skipped_forks_stand_in_no_ones_way(n):
    """A pair that is skipped, for a -1 or a sequence that there is not, does not take its destination from another one."""
    sequences, ps = 2 * n, 16
    pages, table, lens, refs, o = _pool(8 * sequences, ps, sequences, 6, n, (1,), 1)
    g = _gen(27)
    src, dst = torch.randint(0, n, (n,), generator=g).tolist(), list(range(n, 2 * n))
    skipped = [-1] * n
    assert S.fork_sequences(pages, table, lens, refs, _i32(*src, *skipped), _i32(*dst, *dst)).tolist() == [True] * n + [False] * n
    assert _status() == 0
    assert o.fork(src + skipped, dst + dst) == [True] * n + [False] * n
    _same(pages, table, lens, refs, o)
    skipped = [sequences] * n
    assert S.fork_sequences(pages, table, lens, refs, _i32(*src, *skipped), _i32(*dst, *dst)).tolist() == o.fork(src + skipped, dst + dst)
    assert _status() == 4
    _same(pages, table, lens, refs, o)


@pytest.mark.parametrize("chunks", [None, [1, 1, 1, 1], [3, 2, 20, 0]])
@pytest.mark.parametrize("rotated", [False, True])
def test_append_to_sequences_that_were_not_served(chunks, rotated):
    """A sequence that the pool had no room for keeps what it holds, and so does one that shares its pages; a captured step too."""
    ps, H, D = 16, 2, 64
    ragged = chunks is not None
    kv = torch.randn(2, 5, H, ps, D, generator=_gen(28)).to(BF).cuda()
    table, lens, refs = torch.full((4, 3), -1, dtype=torch.int32).cuda(), _i32(0, 0, 0, 0), torch.zeros(5, dtype=torch.int32).cuda()
    assert S.allocate_pages(table, lens, refs, _i32(2 * ps, 0, 5, ps), ps).all()                       # 4 of 5 pages
    assert S.fork_sequences(kv, table, lens, refs, _i32(0), _i32(1)).all()                             # ends with a page: shared
    new = _i32(*(chunks or [1] * 4))
    cut = _i32(*_cu(chunks)) if ragged else None
    T = sum(chunks) if ragged else 4
    g = _gen(29)
    q, k, v = (torch.randn(T, h, D, generator=g).to(BF).cuda() for h in (4, H, H))
    freq = S.rotary_frequencies(D)[0] if rotated else None
    ops.device_status_word(q.device)
    table0, lens0, refs0, kv0 = table.clone(), lens.clone(), refs.clone(), kv.clone()

    def step():
        served = S.allocate_pages(table, lens, refs, new, ps)
        return served, S.append_kv(k, v, kv[0], kv[1], table, lens, cut, q=q if rotated else None, frequencies=freq, served=served)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    results = []
    for run in (lambda: captured if graph.replay() is None else None, step):
        for a, b in ((table, table0), (lens, lens0), (refs, refs0), (kv, kv0)):
            a.copy_(b)
        served, turned = run()
        results.append((served.clone(), None if turned is None else turned.clone(), kv.clone()))
        got, held = served.tolist(), lens.tolist()
        assert got == ([True, False, True, False] if chunks is None or chunks[2] == 1 else [True, False, False, True])
        want = kv0.cpu()
        for i, (t0, t1) in enumerate(zip(_cu(chunks or [1] * 4)[:-1], _cu(chunks or [1] * 4)[1:])):
            for t in range(t0, t1):
                p = held[i] - (t1 - t)
                if not got[i]:
                    assert not rotated or (turned[t] == 0).all()
                    continue
                page = table[i, p // ps].item()
                want[1, page, :, p % ps] = v[t].cpu()
                want[0, page, :, p % ps] = kv[0, page, :, p % ps].cpu() if rotated else k[t].cpu()
                if rotated:
                    _check_rotary(kv[0, page, :, p % ps], k[t], p * freq.cpu(), False)
                    _check_rotary(turned[t], q[t], p * freq.cpu(), False)
        assert torch.equal(kv.cpu(), want)                             # nothing else was written
    assert torch.equal(results[0][2], results[1][2]) and torch.equal(results[0][0], results[1][0])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_forward_mode(interleaved):
    """The tangent of a dual tensor is turned like its value, with and without a backward graph beside it."""
    import torch.autograd.forward_ad as fw
    g = _gen(30)
    freq = S.rotary_frequencies(48)[0]
    pos = torch.tensor([5, 90_000, 3], dtype=torch.int32)
    phase = pos.double()[:, None] * freq.cpu()
    q, k, tq, tk, w = (torch.randn(2, h, 3, 64, generator=g) for h in (3, 1, 3, 1, 3))
    turn = lambda a, b: S.apply_rotary(a, b, pos.cuda(), freq, interleaved, magnitude=0.75)  # noqa: E731
    with fw.dual_level():
        dual = fw.make_dual(q.cuda(), tq.cuda())
        for a in (turn(dual, None), turn(dual, k.cuda())[0], turn(k.cuda(), dual)[1]):
            value, tangent = fw.unpack_dual(a)
            _check_rotary(value, q, phase, interleaved, 0.75)
            _check_rotary(tangent, tq, phase, interleaved, 0.75)
        assert fw.unpack_dual(turn(dual, k.cuda())[1]).tangent is None
        # both of them, in half the bits, token-major
        dq, dk = (fw.make_dual(x.to(BF).cuda().transpose(1, 2), t.to(BF).cuda().transpose(1, 2)) for x, t in ((q, tq), (k, tk)))
        for a, x in zip(S.apply_rotary(dq, dk, pos.cuda(), freq, interleaved, tensor_layout="NHD"), (tq, tk)):
            _check_rotary(fw.unpack_dual(a).tangent.transpose(1, 2), x.to(BF), phase, interleaved)
        # beside a backward graph: the value's gradient, and the tangent's
        leaf, along = q.cuda().requires_grad_(), tq.cuda().requires_grad_()
        value, tangent = fw.unpack_dual(turn(fw.make_dual(leaf, along), k.cuda())[0])
        _check_rotary(tangent.detach(), tq, phase, interleaved, 0.75)
        _check_rotary(torch.autograd.grad(value, leaf, w.cuda(), retain_graph=True)[0], w, -phase, interleaved, 0.75)
        _check_rotary(torch.autograd.grad(tangent, along, w.cuda())[0], w, -phase, interleaved, 0.75)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("neighbour", [False, True])
def test_maximum_that_moves_far_from_zero(dtype, neighbour):
    """Scores near 2^20 in base 2: what the keys before a larger one weigh is what they weigh beside it, to the bits of their difference.

    The products are whole numbers, so the scores are exact. 2 432 equal keys, then one that is larger by one unit of 11.3 in base 2: the
    old ones weigh 2 432 x 2^-11.3 of it. With `neighbour` another row of the same warp goes beyond 2^20 half way.
    Errors: a probability's rounding to the type eps / 2 of its share and the output's own; exponents of up to 12 in 32 bits, their
    exponentials, and sums of up to 64 + 20 terms in a row: together under 1e-5 of the whole."""
    H, D, ps, n = 148, 64, 64, 2560                                    # a tile for each multiprocessor, so that steps follow each other
    B, scale = 64256.0, 7.84375                                        # 251 x 2^8; scale in base 2 is 11.316
    K, V = torch.zeros(n, D), torch.zeros(n, D)
    K[:, 0], K[n - 128:, 1], K[n - 1, 1] = B, -10.0, 1.0
    V[: n - 128], V[n - 1] = -1.0, 1.0
    K[n // 2:, 2] = 32768.0
    q = torch.zeros(20, H, D)
    q[..., :2] = 1.0
    if neighbour:
        q[5, :, 2] = 8.0
    c = dict(seq_lens=_i32(n), page_table=torch.arange(n // ps, dtype=torch.int32).cuda()[None])
    for name, x in (("k_pages", K), ("v_pages", V)):
        c[name] = x.view(n // ps, 1, ps, D).expand(-1, H, -1, -1).contiguous().to(dtype).cuda()
    out, lse = S.paged_attention(q.to(dtype).cuda(), **c, cu_seqlens=_i32(0, 20), max_chunk=20, is_causal=False, scale=scale, return_lse=True)
    x = q[:, 0].double() @ K.double().T * scale
    p = torch.softmax(x, -1)
    want, weight = p @ V.double(), p @ V.double().abs()
    room = torch.finfo(dtype).eps / 2 * (want.abs() + weight) * 1.01 + 1e-5 + (2.0 ** -25 * (1 + n) if dtype == HF else 0.0)
    off = (out.cpu().double() - want[:, None]).abs() - room[:, None]
    assert (off <= 0).all(), off.max()
    assert ((lse.cpu().double() - torch.logsumexp(x, -1)[:, None]).abs() <= 2.0 ** -21 * x.abs().max()).all()
