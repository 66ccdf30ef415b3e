"""Attention, rotary positions and the frame norm on the GPU against 64-bit forms, element by element within derived bounds
(tests/attention_cases.py), at the sizes, masks, strides and types where they can go wrong; and used together."""
import math

import pytest
import torch

import attention_cases as ref
from speech_amd._lib import CtnError
from speech_amd.functional import LinearFn
from speech_amd.modules.attention import RotaryPositions, SelfAttention, attention, rotary_turns, rotate
from speech_amd.modules.norm import FrameLayerNorm, frame_layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def normal(shape, seed, dtype=F32, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std + mean).to(dtype)


# ------------------------------------------------------------------------------------------------ frame norm
NORM_SHAPES = [(1, 1), (1, 64), (7, 3), (1000, 64), (33, 8), (5, 17), (129, 100), (64, 255), (40, 256), (31, 257), (9, 512),
               (17, 1000), (5, 1024), (6, 1025), (3, 2048), (4, 4096), (3, 4097), (2, 8191), (2, 8192), (1, 16384), (2, 16383)]


@pytest.mark.parametrize("dtype,param", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("R,C", NORM_SHAPES)
def test_frame_norm(R, C, dtype, param):
    x, dy = normal((R, C), 1, dtype, 1.5, 0.3), normal((R, C), 2, dtype)
    gamma, beta = normal((C,), 3, param, 0.1, 1.0), normal((C,), 4, param, 0.1)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, gamma, beta)]
    y = frame_layer_norm(*leaves, eps=1e-6)
    y.backward(dy.to(DEV))
    want, bound = ref.frame_norm(x, gamma, beta, 1e-6, dy)
    for n, a, b, t in zip(("y", "dx", "dgamma", "dbeta"), [y] + [l.grad for l in leaves], want, bound):
        ref.check(a, b, t, n)


@pytest.mark.parametrize("R,C", [(5000, 32), (70000, 64), (3001, 200)])
def test_frame_norm_many_rows_same_bits(R, C):
    x, dy = normal((R, C), 1, F32, 1.5, 0.3), normal((R, C), 2)
    gamma, beta = normal((C,), 3, F32, 0.1, 1.0), normal((C,), 4, F32, 0.1)

    def run():
        leaves = [t.to(DEV).requires_grad_(True) for t in (x, gamma, beta)]
        y = frame_layer_norm(*leaves)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy.to(DEV)))

    first = run()
    want, bound = ref.frame_norm(x, gamma, beta, 1e-12, dy)
    for n, a, b, t in zip(("y", "dx", "dgamma", "dbeta"), first, want, bound):
        ref.check(a, b, t, n)
    assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_frame_norm_views_shapes_and_missing_parameters():
    base = normal((6, 5, 50), 5).to(DEV)
    x = base[:, 1:4, 3:40]                                   # rows of 37 of 50, not 16-byte aligned
    y = frame_layer_norm(x, None, None, 1e-6)
    ones, zeros = torch.ones(37), torch.zeros(37)
    want, bound = ref.frame_norm(x.cpu().reshape(-1, 37), ones, zeros, 1e-6)
    assert y.shape == x.shape
    ref.check(y.reshape(-1, 37), want[0], bound[0], "view")
    xt = base.transpose(1, 2).requires_grad_(True)           # features not contiguous
    w = normal((5,), 6).to(DEV).requires_grad_(True)
    y = frame_layer_norm(xt, w, None, 1e-6)
    dy = normal(tuple(y.shape), 7)
    y.backward(dy.to(DEV))
    want, bound = ref.frame_norm(xt.detach().cpu().reshape(-1, 5), w.detach().cpu(), torch.zeros(5), 1e-6, dy.reshape(-1, 5))
    ref.check(y.reshape(-1, 5), want[0], bound[0], "y")
    ref.check(xt.grad.reshape(-1, 5), want[1], bound[1], "dx")
    ref.check(w.grad, want[2], bound[2], "dgamma")
    b = torch.zeros(5, device=DEV, requires_grad=True)       # only the bias wants a gradient
    frame_layer_norm(base.transpose(1, 2), w.detach(), b).backward(dy.to(DEV))
    ref.check(b.grad, want[3], bound[3], "dbeta")
    e = torch.zeros((0, 5), device=DEV, requires_grad=True)
    w.grad = None
    out = frame_layer_norm(e, w, b)
    out.sum().backward()
    assert out.shape == (0, 5) and e.grad.shape == (0, 5) and not w.grad.any()
    # a broadcast gradient (a sum's) has strides of zero
    x2 = normal((9, 5), 8)
    x2d = x2.to(DEV).requires_grad_(True)
    frame_layer_norm(x2d, w, None, 1e-6).sum().backward()
    want, bound = ref.frame_norm(x2, w.detach().cpu(), torch.zeros(5), 1e-6, torch.ones(9, 5))
    ref.check(x2d.grad, want[1], bound[1], "dx of a sum")


def test_frame_norm_constant_rows_are_their_bias():
    """A constant row x has no variance: with eps far below the mean's rounding only the refined mean gives the bias.  The
    first mean is a tree sum of C equal terms, off by d <= (log2 C + 6) f |x|; every element's difference to it is d
    exactly, and what the refinement leaves of d is the rounding of a sum and a division of equal terms, 4 f d at most;
    behind 1 / sqrt(eps) = 1e6 that is 1e6 4 f (log2 C + 6) f |x| (an unrefined mean: 1e6 d, up to the row's whole scale)."""
    for c in (3, 7, 100, 1000):
        x = torch.tensor([1.1, -37.3, 0.0, 1e4])[:, None].expand(4, c).contiguous().to(DEV)
        b = normal((c,), 3).to(DEV)
        y = frame_layer_norm(x, torch.ones(c, device=DEV), b, eps=1e-12)
        bound = 1e6 * 4 * ref.F * (math.log2(c) + 6) * ref.F * x.abs() + 2 * ref.F * b.abs()
        assert ((y - b).abs() <= bound).all(), c


# ------------------------------------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,H,D,R", [(1, 1, 1, 8, 8), (2, 3, 4, 32, 32), (3, 65, 5, 64, 24), (1, 7, 40, 128, 128),
                                       (2, 33, 3, 128, 64), (2, 5, 1, 20, 6), (1, 9, 2, 33, 30), (5, 2, 70, 16, 2),
                                       (4, 6, 2, 10, 0), (1, 300, 2, 256, 256)])
def test_rotary(B, T, H, D, R, interleaved, dtype):
    x, dy = normal((B, T, H, D), 1, dtype), normal((B, T, H, D), 2, dtype)
    turns, _ = rotary_turns(R)
    for positions in (None, torch.arange(T) + 123456, torch.randint(0, 2 ** 31, (B, T), generator=torch.Generator().manual_seed(4))):
        xd = x.to(DEV).requires_grad_(True)
        p = None if positions is None else positions.to(DEV)
        y = rotate(xd, turns.to(DEV), p, offset=11, interleaved=interleaved, magnitude=1.25)
        y.backward(dy.to(DEV))
        pos = torch.arange(T) + 11 if positions is None else positions
        ref.check(y, *ref.rotate(x, turns, pos, interleaved, 1.25), "y")
        ref.check(xd.grad, *ref.rotate(dy, turns, pos, interleaved, 1.25, inverse=True), "dx")


def test_rotary_views_shared_positions_and_orders():
    fused = normal((70, 9, 6, 16), 1)
    turns, _ = rotary_turns(16)
    x = fused.to(DEV)[:, :, 1:5]
    ref.check(rotate(x, turns.to(DEV)), *ref.rotate(fused[:, :, 1:5], turns, torch.arange(9)), "view")
    xt = fused.to(DEV).transpose(1, 2)
    ref.check(rotate(xt, turns.to(DEV)), *ref.rotate(fused.transpose(1, 2), turns, torch.arange(6)), "transposed")
    odd = normal((2, 3, 4, 19), 2).to(DEV)[..., 1:17]        # not 16-byte aligned
    ref.check(rotate(odd, turns.to(DEV)), *ref.rotate(odd.cpu(), turns, torch.arange(3)), "unaligned")
    assert rotate(x[:0], turns.to(DEV)).shape == (0, 9, 4, 16)
    big = normal((1500, 4, 2, 32), 3)                        # batch elements share a block
    t32, _ = rotary_turns(32)
    ref.check(rotate(big.to(DEV), t32.to(DEV), offset=-7), *ref.rotate(big, t32, torch.arange(4) - 7), "many sequences")
    many = torch.zeros((70001, 1, 1, 8), device=DEV)         # more than the grid's second dimension
    many[..., 0] = torch.arange(70001, device=DEV)[:, None, None].float()
    t8, _ = rotary_turns(8)
    assert torch.equal(rotate(many, t8.to(DEV))[..., 0, 0, 0], many[..., 0, 0, 0])      # position 0 turns nothing


def test_rotary_module_keeps_its_frequencies_through_casts():
    m = RotaryPositions(32, scaling=('ramp', 8.0, 4096, 1.0, 32.0)).to(DEV).to(BF16)
    turns, magnitude = rotary_turns(32, scaling=('ramp', 8.0, 4096, 1.0, 32.0))
    assert torch.equal(m.turns.cpu(), turns) and not m.state_dict()
    x = normal((2, 5, 3, 32), 1, BF16)
    ref.check(m(x.to(DEV), offset=10 ** 6), *ref.rotate(x, turns, torch.arange(5) + 10 ** 6, False, magnitude), "module")


# ------------------------------------------------------------------------------------------------ attention
#         B, Tq,  Tk,  H, Hk, D, causal, lengths
ATTENTION = [
    (1, 1, 1, 1, 1, 8, False, None),
    (2, 3, 3, 2, 1, 16, True, None),
    (1, 31, 31, 2, 2, 32, False, None),
    (2, 32, 32, 1, 1, 32, True, None),
    (1, 33, 65, 2, 2, 24, True, None),
    (3, 64, 64, 2, 2, 32, False, [64, 1, 0]),
    (1, 63, 129, 4, 2, 40, True, None),
    (2, 100, 100, 4, 4, 32, False, [77, 100]),
    (1, 128, 127, 2, 1, 64, True, None),
    (1, 130, 50, 2, 2, 64, True, None),                 # the first 80 queries see nothing
    (2, 250, 250, 2, 2, 32, False, None),
    (1, 257, 257, 3, 1, 72, True, [200]),
    (2, 96, 160, 2, 2, 128, False, [160, 33]),
    (1, 200, 200, 4, 2, 128, True, None),
    (1, 513, 513, 2, 1, 48, True, None),
    (2, 5, 700, 6, 2, 104, True, [700, 350]),
    (1, 40, 1, 2, 2, 32, False, None),
    (1, 1, 300, 8, 2, 128, False, None),
]


def run_attention(q, k, v, do, lengths, causal, scale=None):
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    o = attention(*leaves, lengths=lengths, causal=causal, scale=scale)
    return [o.detach()] + list(torch.autograd.grad(o, leaves, do.to(DEV)))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,D,causal,lengths", ATTENTION)
def test_attention(B, Tq, Tk, H, Hk, D, causal, lengths, dtype):
    q, do = normal((B, Tq, H, D), 1, dtype), normal((B, Tq, H, D), 4, dtype)
    k, v = normal((B, Tk, Hk, D), 2, dtype), normal((B, Tk, Hk, D), 3, dtype)
    lens = None if lengths is None else torch.tensor(lengths)
    got = run_attention(q, k, v, do, None if lens is None else lens.to(DEV), causal)
    want, bound = ref.attention(q, k, v, lens, causal, do=do)
    for n, a, b, t in zip(("o", "dq", "dk", "dv"), got, want, bound):
        ref.check(a, b, t, n)
    again = run_attention(q, k, v, do, None if lens is None else lens.to(DEV, torch.int32), causal)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,D,causal,lengths", [
    (1, 1, 5000, 2, 1, 64, False, None), (2, 1, 4100, 8, 2, 128, False, [4100, 7]), (3, 1, 3001, 4, 4, 32, False, [0, 3001, 64]),
    (1, 4, 2500, 8, 2, 96, True, None), (1, 2, 1029, 32, 1, 8, True, [600]), (1, 60, 3000, 1, 1, 128, True, None)])
def test_attention_split_over_keys(B, Tq, Tk, H, Hk, D, causal, lengths, dtype):
    q, k, v = (normal((B, t, h, D), i, dtype) for i, (t, h) in enumerate(((Tq, H), (Tk, Hk), (Tk, Hk))))
    lens = None if lengths is None else torch.tensor(lengths)
    # a cache: head by head, more room than tokens
    kc, vc = (torch.zeros((B, Hk, Tk + 24, D), dtype=dtype, device=DEV) for _ in range(2))
    kc[:, :, :Tk], vc[:, :, :Tk] = k.transpose(1, 2).to(DEV), v.transpose(1, 2).to(DEV)
    o = attention(q.to(DEV), kc[:, :, :Tk].transpose(1, 2), vc[:, :, :Tk].transpose(1, 2),
                  None if lens is None else lens.to(DEV), causal)
    want, bound = ref.attention(q, k, v, lens, causal)
    ref.check(o, want[0], bound[0], "o")
    do = normal((B, Tq, H, D), 9, dtype)
    got = run_attention(q, k, v, do, None if lens is None else lens.to(DEV), causal)
    want, bound = ref.attention(q, k, v, lens, causal, do=do)
    for n, a, b, t in zip(("o", "dq", "dk", "dv"), got, want, bound):
        ref.check(a, b, t, n)


#         B, Tq,  Tk,  H, Hk, D, causal, ragged
MANY = [(1024, 33, 33, 1, 1, 32, False, False), (300, 40, 40, 8, 4, 32, True, True), (520, 20, 70, 2, 2, 8, True, True),
        (520, 70, 20, 2, 2, 24, True, False), (260, 150, 150, 4, 4, 32, True, True), (128, 40, 300, 16, 8, 16, True, True),
        (1024, 1, 129, 1, 1, 32, False, True), (128, 129, 257, 8, 8, 32, False, False), (1030, 5, 3, 1, 1, 16, True, False),
        (512, 100, 40, 4, 2, 64, True, True), (256, 33, 200, 4, 4, 56, False, True), (1024, 35, 300, 2, 1, 40, True, True)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,D,causal,ragged", MANY)
def test_attention_of_many_sequences(B, Tq, Tk, H, Hk, D, causal, ragged, dtype):
    """Enough (sequence, key head) pairs for the backward pass that gives each one a block, within one key block and over
    several, lengths of zero among them."""
    fused = normal((B, max(Tq, Tk), H + 2 * Hk, D), 1, dtype)
    q, k, v = fused[:, :Tq, :H], fused[:, :Tk, H:H + Hk], fused[:, :Tk, H + Hk:]
    do = normal((B, Tq, H, D), 4, dtype)
    lens = None
    if ragged:
        lens = torch.randint(0, Tk + 1, (B,), generator=torch.Generator().manual_seed(5))
        lens[:2] = torch.tensor([0, Tk])
        for b in range(B):
            fused[b, lens[b]:, H:] = math.nan if b % 2 else math.inf
    fd = fused.to(DEV)
    leaves = [fd[:, :Tq, :H].requires_grad_(True), fd[:, :Tk, H:H + Hk].requires_grad_(True),
              fd[:, :Tk, H + Hk:].requires_grad_(True)]

    def run():
        o = attention(*leaves, lengths=None if lens is None else lens.to(DEV), causal=causal)
        return [o.detach()] + list(torch.autograd.grad(o, leaves, do.to(DEV)))

    got = run()
    want, bound = ref.attention(q, k, v, lens, causal, do=do)
    for n, a, b, t in zip(("o", "dq", "dk", "dv"), got, want, bound):
        ref.check(a, b, t, n)
    assert all(torch.equal(a, b) for a, b in zip(got, run()))


#          B, Tq,  Tk,  H, Hk, D, causal, ragged
SHORT = [(2, 96, 128, 4, 2, 32, True, True), (1, 97, 128, 4, 2, 32, True, False), (3, 192, 100, 2, 2, 24, False, True),
         (3, 193, 100, 2, 2, 24, False, True), (2, 64, 250, 2, 2, 32, True, True), (1, 1, 700, 1, 1, 8, False, True),
         (96, 150, 150, 4, 4, 32, True, True), (95, 150, 150, 4, 4, 32, False, False)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,D,causal,ragged", SHORT)
def test_attention_of_short_sequences(B, Tq, Tk, H, Hk, D, causal, ragged, dtype):
    """Both sides of the rules that give a key head's gradients to one block: six stages of 128 keys by 32 queries and seven, 384
    key heads and fewer."""
    q, do = normal((B, Tq, H, D), 1, dtype), normal((B, Tq, H, D), 2, dtype)
    k, v = normal((B, Tk, Hk, D), 3, dtype), normal((B, Tk, Hk, D), 4, dtype)
    lens = None
    if ragged:
        lens = torch.randint(0, Tk + 1, (B,), generator=torch.Generator().manual_seed(7))
        lens[0] = Tk - 1
        for b in range(B):
            k[b, lens[b]:] = math.nan
            v[b, lens[b]:] = math.inf
    on = None if lens is None else lens.to(DEV)
    got = run_attention(q, k, v, do, on, causal)
    want, bound = ref.attention(q, k, v, lens, causal, do=do)
    for n, a, b, t in zip(("o", "dq", "dk", "dv"), got, want, bound):
        ref.check(a, b, t, n)


#         B, Tq,  Tk,  H, Hk, D, causal, ragged
WIDE = [(3, 300, 300, 6, 2, 128, True, True), (2, 65, 700, 2, 2, 72, False, True), (1, 1100, 1100, 2, 1, 120, True, False),
        (2, 40, 64, 4, 1, 96, True, True), (9, 130, 20, 8, 8, 128, False, True), (1, 33, 129, 3, 3, 104, True, True)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,D,causal,ragged", WIDE)
def test_attention_of_wide_heads(B, Tq, Tk, H, Hk, D, causal, ragged, dtype):
    """Heads of more than 64 features, whose gradients are formed by pairs of waves: one pair a block, two and four, the walk
    over queries cut and not, tiles that end inside the sequences."""
    q, do = normal((B, Tq, H, D), 1, dtype), normal((B, Tq, H, D), 2, dtype)
    k, v = normal((B, Tk, Hk, D), 3, dtype), normal((B, Tk, Hk, D), 4, dtype)
    lens = None
    if ragged:
        lens = torch.randint(0, Tk + 1, (B,), generator=torch.Generator().manual_seed(6))
        lens[0] = Tk - 1
        for b in range(B):
            k[b, lens[b]:] = math.nan
            v[b, lens[b]:] = math.inf
    on = None if lens is None else lens.to(DEV)
    got = run_attention(q, k, v, do, on, causal)
    want, bound = ref.attention(q, k, v, lens, causal, do=do)
    for n, a, b, t in zip(("o", "dq", "dk", "dv"), got, want, bound):
        ref.check(a, b, t, n)
    assert all(torch.equal(a, b) for a, b in zip(got, run_attention(q, k, v, do, on, causal)))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,H,Hk,D", [(2, 200, 2, 2, 128), (1, 700, 4, 1, 48), (600, 140, 2, 2, 32)])
def test_single_gradients_are_those_of_all(B, T, H, Hk, D, dtype):
    """Every subset of the three gradients has the bits it has when all are asked for."""
    q, do = normal((B, T, H, D), 1, dtype).to(DEV), normal((B, T, H, D), 2, dtype).to(DEV)
    k, v = normal((B, T, Hk, D), 3, dtype).to(DEV), normal((B, T, Hk, D), 4, dtype).to(DEV)

    def run(want):
        leaves = [t.clone().requires_grad_(w) for t, w in zip((q, k, v), want)]
        attention(*leaves, causal=True).backward(do)
        return [t.grad for t in leaves]

    every = run((True, True, True))
    for n in range(1, 7):
        want = [bool(n & 1), bool(n & 2), bool(n & 4)]
        for g, e, w in zip(run(want), every, want):
            assert torch.equal(g, e) if w else g is None


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_reads_nothing_behind_a_length(dtype):
    q, k, v, do = (normal((2, 50, 2, 32), i, dtype) for i in range(4))
    lens = torch.tensor([20, 0])
    kn, vn = k.clone(), v.clone()
    for b in range(2):
        kn[b, lens[b]:], vn[b, lens[b]:] = math.nan, math.inf
    for causal in (False, True):
        got = run_attention(q, kn, vn, do, lens.to(DEV), causal)
        want, bound = ref.attention(q, k, v, lens, causal, do=do)
        for n, a, b, t in zip(("o", "dq", "dk", "dv"), got, want, bound):
            ref.check(a, b, t, n)
        assert not got[0][1].any() and not got[2][0, 20:].any() and not got[3][1].any()
    out_of_range = torch.tensor([-3, 1000], device=DEV)      # clamped to 0 and Tk
    want, bound = ref.attention(q, k, v, torch.tensor([0, 50]))
    ref.check(attention(q.to(DEV), k.to(DEV), v.to(DEV), out_of_range), want[0], bound[0], "lengths out of range")
    ref.check(attention(q.to(DEV), k.to(DEV), v.to(DEV), out_of_range.int()), want[0], bound[0], "lengths out of range")


def test_attention_views_orders_and_shared_heads():
    fused = normal((3, 40, 8, 32), 1)
    do = normal((3, 40, 4, 32), 2)
    fd = fused.to(DEV).requires_grad_(True)
    o = attention(fd[:, :, :4], fd[:, :, 4:6], fd[:, :, 6:], causal=True)
    o.backward(do.to(DEV))
    want, bound = ref.attention(fused[:, :, :4], fused[:, :, 4:6], fused[:, :, 6:], causal=True, do=do)
    ref.check(o, want[0], bound[0], "o")
    ref.check(fd.grad, torch.cat(want[1:], 2), torch.cat(bound[1:], 2), "gradient of the fused projection")
    # one key / value sequence for the whole batch: the broadcast's gradient adds up over it
    q, k = normal((3, 20, 2, 16), 3), normal((1, 33, 2, 16), 4)
    kd = k.to(DEV).requires_grad_(True)
    o = attention(q.to(DEV), kd.expand(3, -1, -1, -1), kd.expand(3, -1, -1, -1))
    do = normal((3, 20, 2, 16), 5)
    o.backward(do.to(DEV))
    want, bound = ref.attention(q, k.expand(3, -1, -1, -1), k.expand(3, -1, -1, -1), do=do)
    ref.check(kd.grad, (want[2] + want[3]).sum(0, keepdim=True), (bound[2] + bound[3]).sum(0, keepdim=True) * (1 + 1e-5) +
              4 * ref.F * (want[2].abs() + want[3].abs()).sum(0, keepdim=True), "shared keys")
    # features not contiguous, unaligned
    qt = normal((2, 16, 3, 10), 6).to(DEV).transpose(1, 3)
    un = normal((2, 10, 3, 17), 7).to(DEV)[..., 1:]
    want, bound = ref.attention(qt.cpu(), un.cpu(), un.cpu())
    ref.check(attention(qt, un, un), want[0], bound[0], "orders")
    want, bound = ref.attention(qt.cpu(), un.cpu(), un.cpu(), scale=0.7)
    ref.check(attention(qt, un, un, scale=0.7), want[0], bound[0], "scale")


def test_attention_without_queries_keys_or_batch():
    z = lambda *s: torch.zeros(s, device=DEV, requires_grad=True)
    q, k = normal((2, 5, 2, 8), 1).to(DEV).requires_grad_(True), z(2, 0, 2, 8)
    o = attention(q, k, k)
    o.sum().backward()
    assert not o.any() and not q.grad.any() and k.grad.shape == (2, 0, 2, 8)
    q, k = z(2, 0, 2, 8), normal((2, 5, 2, 8), 1).to(DEV).requires_grad_(True)
    o = attention(q, k, k)
    o.sum().backward()
    assert o.shape == (2, 0, 2, 8) and not k.grad.any()
    assert attention(z(0, 4, 2, 8), z(0, 4, 2, 8), z(0, 4, 2, 8)).shape == (0, 4, 2, 8)


def test_attention_large_scores_and_far_rows():
    q, k, v, do = (normal((1, 70, 1, 32), i) for i in range(4))
    q = q * 30                                               # probabilities of zero and one
    got = run_attention(q, k, v, do, None, False)
    want, bound = ref.attention(q, k, v, None, False, do=do)
    for n, a, b, t in zip(("o", "dq", "dk", "dv"), got, want, bound):
        ref.check(a, b, t, n)
    # a cache whose heads lie more than 2^31 elements apart
    cache = torch.empty((2, 2 ** 31 + 64), dtype=BF16, device=DEV)
    kv = cache[:, -64 * 32:].view(2, 64, 32)
    kb = normal((64, 2, 32), 5, BF16)
    kv.copy_(kb.transpose(0, 1))
    k4 = kv.transpose(0, 1)[None]                            # (1, 64, 2, 32)
    qb = normal((1, 3, 2, 32), 6, BF16)
    want, bound = ref.attention(qb, kb[None], kb[None])
    ref.check(attention(qb.to(DEV), k4, k4), want[0], bound[0], "far heads")


def test_attention_gradient_against_differences():
    q, k, v, do = (normal((2, 37, 2, 16), i) for i in range(4))
    got = run_attention(q, k, v, do, None, True)
    for i, g in enumerate(got[1:]):
        d = normal((2, 37, 2, 16), 10 + i)
        h = 2.0 ** -6
        f = []
        for sgn in (1, -1):
            x = [q, k, v]
            x[i] = x[i] + sgn * h * d
            o = attention(*[t.to(DEV) for t in x], causal=True)
            f.append((o.double().cpu() * do.double()).sum().item())
        diff, grad = (f[0] - f[1]) / (2 * h), (g.double().cpu() * d.double()).sum().item()
        # third derivatives of order one along a direction of norm sqrt(n): h^2 n / 6; fp32 outputs: f n / h
        assert abs(diff - grad) <= h * h * q.numel() / 6 + ref.F * q.numel() / h, (i, diff, grad)


# ------------------------------------------------------------------------------------------------ together
def unit(x, norm, att, w):
    return att(norm(x)) @ w


def test_norm_projection_rotary_attention_together():
    """The attention form of a dual-path unit up to its output projection against its formula in 64 bits; everything between
    is fp32, so 2e-5 of the largest entry as for every fp32 kernel of the framework (the gradients: 1e-4)."""
    torch.manual_seed(0)
    norm, att = FrameLayerNorm(24).to(DEV), SelfAttention(24, 32, 2, causal=True).to(DEV)
    with torch.no_grad():
        norm.weight.copy_(normal((24,), 3, std=0.1, mean=1.0))
        norm.bias.copy_(normal((24,), 4, std=0.1))
    x = normal((3, 50, 24), 1)
    dy = normal((3, 50, 32), 2)
    xd = x.to(DEV).requires_grad_(True)
    y = att(norm(xd))
    y.backward(dy.to(DEV))
    params = {n: p.detach().cpu().double().requires_grad_(True) for n, p in
              list(norm.named_parameters()) + list(att.named_parameters())}
    x64 = x.double().requires_grad_(True)
    z = torch.nn.functional.layer_norm(x64, (24,), params["weight"], params["bias"], 1e-12)
    qkv = (z @ params["in_proj.weight"].t() + params["in_proj.bias"]).view(3, 50, 6, 16)
    turns, _ = rotary_turns(16)
    ang = torch.arange(50).double()[:, None] * turns * 2 * math.pi
    c, s = torch.cos(ang)[None, :, None], torch.sin(ang)[None, :, None]
    a, b = qkv[:, :, :4, :8], qkv[:, :, :4, 8:]
    qk = torch.cat((a * c - b * s, a * s + b * c), -1)
    q, k, v = qk[:, :, :2].transpose(1, 2), qk[:, :, 2:].transpose(1, 2), qkv[:, :, 4:].transpose(1, 2)
    sc = (q @ k.transpose(2, 3) / 4).masked_fill(~torch.ones(50, 50, dtype=torch.bool).tril(), -math.inf)
    y64 = (torch.softmax(sc, 3) @ v).transpose(1, 2).reshape(3, 50, 32)
    y64.backward(dy.double())

    def rel(p, r):
        return ((p.detach().cpu().double() - r).abs().max() / r.abs().max()).item()

    assert rel(y, y64.detach()) < 2e-5
    assert rel(xd.grad, x64.grad) < 1e-4
    for n, p in list(norm.named_parameters()) + list(att.named_parameters()):
        assert rel(p.grad, params[n].grad) < 1e-4, n


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,T,causal,D", [(3, 45, True, 16), (600, 45, False, 16), (3, 45, False, 24), (520, 150, True, 32),
                                          (2, 300, True, 80)])
def test_fused_projection_equals_its_parts(N, T, causal, D, dtype):
    """RotarySelfAttentionFn runs the very kernels that rotate and attention run on the parts: the same bits."""
    from speech_amd.functional import RotarySelfAttentionFn
    H = 2
    turns = rotary_turns(D)[0].to(DEV)
    qkv, do = normal((N, T, 3 * H, D), 1, dtype).to(DEV), normal((N, T, H, D), 2, dtype).to(DEV)
    lens = torch.randint(0, T + 1, (N,), generator=torch.Generator().manual_seed(1)).to(DEV)
    a = qkv.clone().requires_grad_(True)
    ya = RotarySelfAttentionFn.apply(a, turns, N == 3, 1.5, lens, causal)
    ya.backward(do)
    b = qkv.clone().requires_grad_(True)
    qk = rotate(b[:, :, :2 * H], turns, interleaved=N == 3, magnitude=1.5)
    yb = attention(qk[:, :, :H], qk[:, :, H:], b[:, :, 2 * H:], lens, causal)
    yb.backward(do)
    assert torch.equal(ya, yb) and torch.equal(a.grad, b.grad)


def test_self_attention_takes_its_rotary_module_as_it_is():
    """Another layout, part of a head and a scaling, put into the module: the output is that of its parts."""
    torch.manual_seed(1)
    m = SelfAttention(24, 64, num_heads=2, causal=True).to(DEV)
    m.rotary = RotaryPositions(32, rotary_dim=16, interleaved=True, scaling=('ramp', 4.0, 512, 1, 32)).to(DEV)
    x = normal((2, 37, 24), 3).to(DEV)
    with torch.no_grad():
        qkv = LinearFn.apply(x, m.in_proj.weight, m.in_proj.bias).view(2, 37, 6, 32)
        qk = m.rotary(qkv[:, :, :4])
        want = attention(qk[:, :, :2], qk[:, :, 2:], qkv[:, :, 4:], causal=True).view(2, 37, 64)
        assert torch.equal(m(x), want)
    assert torch.equal(m(x), want)


def test_second_derivatives_are_refused():
    """autograd.grad calls x unreachable from its gradient, backward() names the reason: an error either way."""
    x = normal((4, 9, 2, 16), 1).to(DEV).requires_grad_(True)
    turns = rotary_turns(16)[0].to(DEV)
    for f in (lambda t: attention(t, t, t), lambda t: rotate(t, turns), lambda t: frame_layer_norm(t)):
        g, = torch.autograd.grad(f(x).square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="not have been used"):
            torch.autograd.grad(g.sum(), x)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


def test_other_types_are_refused():
    turns = rotary_turns(16)[0].to(DEV)
    for dtype in (torch.float16, torch.float64):
        x = torch.zeros((1, 2, 2, 16), device=DEV, dtype=dtype)
        for f in (lambda: attention(x, x, x), lambda: rotate(x, turns), lambda: frame_layer_norm(x)):
            with pytest.raises(CtnError, match="float32 or bfloat16"):
                f()
    x = torch.zeros((1, 2, 2, 16), device=DEV)
    for f in (lambda: frame_layer_norm(x, torch.ones(16, device=DEV, dtype=BF16)), lambda: frame_layer_norm(x, torch.ones(15, device=DEV)),
              lambda: frame_layer_norm(x, torch.ones(16)), lambda: rotate(x, turns.cpu()), lambda: rotate(x, turns.float()),
              lambda: rotate(x, rotary_turns(18)[0].to(DEV)), lambda: rotate(x[0], turns),
              lambda: rotate(x, turns, torch.zeros(3, device=DEV, dtype=torch.int64)),
              lambda: rotate(x, turns, torch.zeros(2, device=DEV)), lambda: rotate(x, turns, torch.arange(2)),
              lambda: attention(x, x, x, lengths=torch.tensor([1])), lambda: attention(x, x, x, scale=0.0),
              lambda: frame_layer_norm(torch.zeros((1, 16385), device=DEV)), lambda: frame_layer_norm(x, eps=-1.0)):
        with pytest.raises(CtnError):
            f()


def test_captured_steps_replay_like_eager_ones():
    """Norm, rotary and attention with their gradients in one graph: every replay on new inputs equals the eager pass, with
    eager work in between; a second graph has its own workspaces."""
    turns = rotary_turns(32)[0].to(DEV)
    shapes = [(2, 90, 2, 32), (1, 3, 2, 32)]
    caches = [normal((2, 90, 2, 32), 8).to(DEV), normal((1, 4000, 2, 32), 9).to(DEV)]     # the second is split over keys

    def step(x, k, w):
        y = frame_layer_norm(x, w, None)
        y = rotate(y, turns, offset=5)
        o = attention(y, k, k, causal=True)
        return (o,) + torch.autograd.grad(o, (x, k, w), torch.ones_like(o))

    graphs = []
    for i in range(2):
        x = normal(shapes[i], 1).to(DEV).requires_grad_(True)
        k = caches[i].clone().requires_grad_(True)
        w = torch.ones(32, device=DEV, requires_grad=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, k, w)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(x, k, w)
        graphs.append((g, x, k, w, out))
    for n in range(4):
        for i, (g, x, k, w, out) in enumerate(graphs):
            with torch.no_grad():
                x.copy_(normal(shapes[i], 20 + n))
            g.replay()
        for i, (g, x, k, w, out) in enumerate(graphs):
            eager = step(*[t.detach().clone().requires_grad_(True) for t in (x, k, w)])
            torch.cuda.synchronize()
            for a, b in zip(out, eager):
                assert torch.equal(a, b)


def test_captured_module_with_lengths_replays_like_eager():
    """SelfAttention and its input's gradient in a graph; inputs and lengths change between the replays."""
    torch.manual_seed(2)
    m = SelfAttention(24, 64, num_heads=2).to(DEV)
    x = normal((3, 50, 24), 1).to(DEV).requires_grad_(True)
    lens = torch.tensor([50, 7, 0], device=DEV)

    def step(x, lens):
        o = m(x, lens)
        return (o.detach(),) + torch.autograd.grad(o, (x,), torch.ones_like(o))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, lens)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(x, lens)
    for n in range(3):
        with torch.no_grad():
            x.copy_(normal((3, 50, 24), 10 + n))
            lens.copy_(torch.tensor([n, 50 - n, 33]))
        g.replay()
        eager = step(x.detach().clone().requires_grad_(True), lens.clone())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_two_threads_on_two_streams():
    """Calls from two threads at once, each on a stream of its own: the same bits as alone."""
    import threading
    cases = [(normal((2, 150, 4, 32), 1), normal((2, 150, 4, 32), 2)), (normal((3, 90, 2, 128), 3, BF16), normal((3, 90, 2, 128), 4, BF16))]
    base = [run_attention(q, q, q, do, None, True) for q, do in cases]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(8):
                    q, do = cases[i]
                    got[i].append(run_attention(q, q, q, do, None, True))
                    frame_layer_norm(q.to(DEV))
            stream.synchronize()
        except Exception as e:                               # an error in a thread would otherwise pass unseen
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for i in range(2):
        assert len(got[i]) == 8 and all(torch.equal(a, b) for r in got[i] for a, b in zip(r, base[i]))


def test_calls_on_a_side_stream():
    side = torch.cuda.Stream()
    q, k, v, do = (normal((2, 300, 4, 32), i) for i in range(4))
    base = run_attention(q, k, v, do, None, False)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [run_attention(q, k, v, do, None, False) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, base))


@pytest.mark.parametrize("causal", [False, True])
def test_dual_path_network_with_attention(causal):
    """DPRNN-TasNet in its attention form: the separator's dual-path stack against the formula in 64 bits (through torch's own
    operations on the CPU), gradients included; a causal stack's output does not depend on later chunks."""
    from speech_amd.models.dprnn import DPRNN
    torch.manual_seed(1)
    net = DPRNN(16, 32, num_blocks=2, causal=causal, rnn_type='attention', num_heads=2).to(DEV)
    x, dy = normal((2, 16, 7, 10), 1), normal((2, 16, 7, 10), 2)
    xd = x.to(DEV).requires_grad_(True)
    y = net(xd)
    y.backward(dy.to(DEV))
    params = {n: p.detach().cpu().double().requires_grad_(True) for n, p in net.named_parameters()}
    x64 = x.double().requires_grad_(True)
    turns, _ = rotary_turns(16)

    def path(z, name, walk, mask):
        P = {n: params[name + "." + n] for n in ("norm1d.weight", "norm1d.bias", "attention.in_proj.weight",
                                                 "attention.in_proj.bias", "fc.weight", "fc.bias")}
        r = z.permute(0, 3, 2, 1) if walk else z.permute(0, 2, 3, 1)
        h = torch.nn.functional.layer_norm(r, (16,), P["norm1d.weight"], P["norm1d.bias"], 1e-12)
        qkv = (h @ P["attention.in_proj.weight"].t() + P["attention.in_proj.bias"]).unflatten(-1, (6, 16))
        T = r.shape[2]
        ang = torch.arange(T).double()[:, None] * turns * 2 * math.pi
        c, s = torch.cos(ang)[None, None, :, None], torch.sin(ang)[None, None, :, None]
        a, b = qkv[..., :4, :8], qkv[..., :4, 8:]
        qk = torch.cat((a * c - b * s, a * s + b * c), -1)
        q, k, v = (t.transpose(2, 3) for t in (qk[..., :2, :], qk[..., 2:, :], qkv[..., 4:, :]))
        sc = q @ k.transpose(-2, -1) / 4
        if mask:
            sc = sc.masked_fill(~torch.ones(T, T, dtype=torch.bool).tril(), -math.inf)
        o = (torch.softmax(sc, -1) @ v).transpose(2, 3).flatten(-2) @ P["fc.weight"].t() + P["fc.bias"]
        return z + (o.permute(0, 3, 2, 1) if walk else o.permute(0, 3, 1, 2))

    z = x64
    for i in range(2):
        z = path(z, "net.%d.intra_chunk_block" % i, False, False)
        z = path(z, "net.%d.inter_chunk_block" % i, True, causal)
    z.backward(dy.double())

    def rel(p, r):
        return ((p.detach().cpu().double() - r).abs().max() / r.abs().max()).item()

    assert rel(y, z.detach()) < 1e-4
    assert rel(xd.grad, x64.grad) < 1e-4
    for n, p in net.named_parameters():
        assert rel(p.grad, params[n].grad) < 1e-4, n
    if causal:
        x2 = x.clone()
        x2[:, :, 4:] += 1
        with torch.no_grad():
            assert torch.equal(net(x2.to(DEV))[:, :, :4], y.detach()[:, :, :4])


def test_dual_path_tasnet_with_attention_trains_a_step():
    from dprnn_cases import SMALL_CAUSAL3
    from speech_amd.criterion.pit import PIT1d
    from speech_amd.criterion.sdr import NegSISDR
    from speech_amd.models.dprnn_tasnet import DPRNNTasNet
    torch.manual_seed(1)
    model = DPRNNTasNet(**dict(SMALL_CAUSAL3, sep_hidden_channels=32, rnn_type='attention')).to(DEV)
    src = (0.1 * normal((2, 3, 250), 1)).to(DEV)
    loss, _ = PIT1d(NegSISDR(), n_sources=3)(model(src.sum(1, keepdim=True)), src)
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    assert all(p.grad.any() for n, p in model.named_parameters() if "in_proj.weight" in n)
