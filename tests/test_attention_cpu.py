"""Refusals of the frame norm, rotary positions and attention, and what their host side computes, without a GPU."""
import ctypes as C
import math

import pytest
import torch

import attention_cases as ref
from speech_amd import _lib, ops
from speech_amd.modules.attention import RotaryPositions, SelfAttention, attention, rotary_turns, rotate
from speech_amd.modules.norm import FrameLayerNorm, frame_layer_norm


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 2, 8)
    for call in (lambda: frame_layer_norm(x), lambda: attention(x, x, x),
                 lambda: rotate(x, rotary_turns(8)[0])):
        with pytest.raises(_lib.CtnError, match="GPU only"):
            call()


class Fake:
    """Stands in for a GPU tensor in the checks that run before any pointer is used."""

    def __init__(self, shape, dtype=torch.float32, device="cuda:0"):
        self.shape, self.dtype, self.is_cuda, self.device = torch.Size(shape), dtype, True, torch.device(device)

    def dim(self):
        return len(self.shape)


@pytest.mark.parametrize("q,k,v,lengths,match", [
    (Fake((2, 3, 4, 12)), Fake((2, 3, 4, 12)), Fake((2, 3, 4, 12)), None, "multiples of 8"),
    (Fake((2, 3, 4, 136)), Fake((2, 3, 4, 136)), Fake((2, 3, 4, 136)), None, "up to 128"),
    (Fake((2, 3, 4, 16)), Fake((2, 3, 3, 16)), Fake((2, 3, 3, 16)), None, "a multiple"),
    (Fake((2, 3, 4, 16)), Fake((2, 3, 0, 16)), Fake((2, 3, 0, 16)), None, "a multiple"),
    (Fake((2, 3, 4, 16)), Fake((2, 5, 4, 16)), Fake((2, 6, 4, 16)), None, "Tk, Hk, D"),
    (Fake((2, 3, 4, 16)), Fake((1, 5, 4, 16)), Fake((1, 5, 4, 16)), None, "Tk, Hk, D"),
    (Fake((2, 3, 4, 16)), Fake((2, 5, 4, 24)), Fake((2, 5, 4, 24)), None, "Tk, Hk, D"),
    (Fake((2, 3, 16)), Fake((2, 5, 16)), Fake((2, 5, 16)), None, "Tk, Hk, D"),
    (Fake((2, 3, 4, 16), torch.float16), Fake((2, 3, 4, 16)), Fake((2, 3, 4, 16)), None, "float32 or bfloat16"),
    (Fake((2, 3, 4, 16)), Fake((2, 3, 4, 16), torch.bfloat16), Fake((2, 3, 4, 16)), None, "one type"),
    (Fake((2, 3, 4, 16)), Fake((2, 3, 4, 16), device="cuda:1"), Fake((2, 3, 4, 16)), None, "tensors on"),
    (Fake((2, 3, 4, 16)), Fake((2, 3, 4, 16)), Fake((2, 3, 4, 16)), Fake((3,), torch.int32), "lengths"),
    (Fake((2, 3, 4, 16)), Fake((2, 3, 4, 16)), Fake((2, 3, 4, 16)), Fake((2,), torch.float32), "lengths"),
])
def test_attention_refusals(q, k, v, lengths, match):
    with pytest.raises(_lib.CtnError, match=match):
        ops.check_attention(q, k, v, lengths)


def good_args(**over):
    a = _lib.AttnArgs()
    a.batch, a.Tq, a.Tk, a.H, a.Hk, a.D, a.type, a.scale = 2, 8, 8, 4, 2, 16, _lib.TYPE_F32, 0.25
    for n in ("q", "k", "v", "o"):
        setattr(a, n, 1 << 20)
        for s, st in zip("bth", (1024, 64, 16)):
            setattr(a, n + "_" + s, st)
    for n, x in over.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("over", [
    dict(type=7), dict(H=3), dict(Hk=0), dict(H=0), dict(D=12), dict(D=0), dict(D=136), dict(scale=0.0), dict(scale=-1.0),
    dict(scale=math.nan), dict(scale=math.inf), dict(batch=-1), dict(Tq=-1), dict(Tk=-1), dict(Tk=2 ** 30), dict(q=None),
    dict(k=None), dict(v=None), dict(o=None), dict(q=(1 << 20) + 4), dict(k_t=2), dict(v_h=6), dict(o_b=1), dict(q_b=-64)])
def test_attention_c_entry_refuses(over):
    lib = _lib.load()
    a = good_args(**over)
    assert lib.ctn_attn_fwd(C.byref(a), None) == -1
    assert b"ctn_attn_fwd" in lib.ctn_last_error()
    assert lib.ctn_attn_fwd_ws_floats(C.byref(a)) == -1 and lib.ctn_attn_bwd_ws_floats(C.byref(a)) == -1
    assert lib.ctn_attn_bwd(C.byref(a), None) == -1


def test_attention_c_entry_wants_its_workspaces_and_gradient():
    lib = _lib.load()
    a = good_args(Tq=1, Tk=10000)
    need = lib.ctn_attn_fwd_ws_floats(C.byref(a))
    assert need > 0
    a.ws, a.ws_floats = 1 << 20, need - 1
    assert lib.ctn_attn_fwd(C.byref(a), None) == -1 and b"workspace" in lib.ctn_last_error()
    bf16 = _lib.TYPE_BF16                      # (short fp32 calls of narrow heads take one launch, without a workspace)
    assert lib.ctn_attn_bwd_ws_floats(C.byref(good_args())) == 0
    b = good_args(type=bf16)
    assert lib.ctn_attn_bwd_ws_floats(C.byref(b)) >= 2 * 4 * 8
    assert lib.ctn_attn_bwd(C.byref(b), None) == -1 and b"lse" in lib.ctn_last_error()
    b = good_args(type=bf16, d_o=1 << 20, lse=1 << 20, do_b=1024, do_t=64, do_h=16)
    assert lib.ctn_attn_bwd(C.byref(b), None) == -1 and b"workspace" in lib.ctn_last_error()
    b = good_args(type=bf16, d_o=1 << 20, lse=1 << 20, do_b=1024, do_t=64, do_h=16, ws=1 << 20, ws_floats=1 << 20, dq=(1 << 20) + 8)
    assert lib.ctn_attn_bwd(C.byref(b), None) == -1 and b"aligned" in lib.ctn_last_error()
    # nothing to do is no error, and needs no pointer
    assert lib.ctn_attn_fwd(C.byref(good_args(batch=0, q=None, k=None, v=None, o=None)), None) == 0
    assert lib.ctn_attn_fwd(C.byref(good_args(Tq=0, q=None, o=None)), None) == 0


def test_norm_and_rotary_c_entries_refuse():
    lib = _lib.load()
    p = 1 << 20
    fwd = lambda **o: lib.ctn_frame_norm_fwd(*[{**dict(x=p, ldx=8, R=4, C=8, t=0, g=p, b=p, w=0, eps=1e-6, y=p, ldy=8, st=p,
                                                       s=None), **o}[n] for n in "x ldx R C t g b w eps y ldy st s".split()])
    for over in (dict(t=5), dict(w=1), dict(C=0), dict(C=16385), dict(R=-1), dict(x=None), dict(y=None), dict(ldy=7),
                 dict(eps=-1.0)):
        assert fwd(**over) == -1, over
    assert fwd(R=0, x=None, y=None) == 0
    bwd = lambda **o: lib.ctn_frame_norm_bwd(*[{**dict(dy=p, ldd=8, x=p, ldx=8, R=4, C=8, t=0, g=p, w=0, st=p, dx=p, lx=8, dg=p,
                                                       db=p, ws=p, n=0, s=None), **o}[n]
                                               for n in "dy ldd x ldx R C t g w st dx lx dg db ws n s".split()])
    for over in (dict(R=400), dict(R=400, ws=None, n=1 << 20), dict(st=None), dict(t=3), dict(lx=7), dict(C=20000)):
        assert bwd(**over) == -1, over
    rot = lambda **o: lib.ctn_rotary(*[{**dict(x=p, xb=64, xt=16, xh=8, B=2, T=4, H=2, D=8, t=0, pos=None, pb=0, first=0, tu=p,
                                               R=8, i=0, inv=0, m=1.0, y=p, yb=64, yt=16, yh=8, s=None), **o}[n]
                                       for n in "x xb xt xh B T H D t pos pb first tu R i inv m y yb yt yh s".split()])
    for over in (dict(t=2), dict(R=7), dict(R=10), dict(R=-2), dict(B=-1), dict(D=0), dict(x=None), dict(y=None), dict(tu=None)):
        assert rot(**over) == -1, over
    assert rot(B=0, x=None, y=None) == 0


def test_rotary_turns_and_scalings():
    t, m = rotary_turns(8)
    assert m == 1.0 and t.dtype == torch.float64
    assert torch.allclose(t * 2 * math.pi, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    assert torch.allclose(rotary_turns(8, scaling=('linear', 4.0))[0], t / 4)
    b = rotary_turns(8, scaling=('base', 4.0))[0]
    assert b[0] == t[0] and torch.allclose(b[-1], t[-1] / 4)
    r, m = rotary_turns(8, scaling=('ramp', 4.0, 1000, 1.0, 100.0))
    n = t * 1000                                             # 159, 15.9, 1.59, 0.159 turns over the trained length
    keep = ((n - 1) / 99).clamp(0, 1)
    assert torch.allclose(r, t * keep + t / 4 * (1 - keep)) and r[0] == t[0] and torch.allclose(r[-1], t[-1] / 4)
    assert m == pytest.approx(0.1 * math.log(4.0) + 1)
    assert rotary_turns(0)[0].numel() == 0
    for bad in (('cubic', 2.0), ('linear', 0.5)):
        with pytest.raises(ValueError, match="scaling"):
            rotary_turns(8, scaling=bad)
    for call in (lambda: rotary_turns(7), lambda: rotary_turns(2, scaling=('base', 2.0)), lambda: RotaryPositions(8, 10),
                 lambda: rotary_turns(8, scaling=('ramp', 2.0, 100, 3.0, 3.0)), lambda: SelfAttention(16, 24, 2),
                 lambda: SelfAttention(16, 512, 2)):
        with pytest.raises(ValueError):
            call()


def test_rotary_frequencies_survive_casts_and_state_dict():
    m = RotaryPositions(16, 8)
    want = rotary_turns(8)[0]
    assert torch.equal(m.to(torch.bfloat16).turns, want) and torch.equal(m.float().turns, want) and not m.state_dict()
    n = FrameLayerNorm(8)
    assert list(n.state_dict()) == ["weight", "bias"]


def test_reference_gradients_against_differences():
    """The 64-bit forms that the GPU tests compare with: their gradients against central differences."""
    g = torch.Generator().manual_seed(1)
    mk = lambda *s: torch.randn(s, generator=g, dtype=torch.float64).float()
    q, k, v, do = mk(2, 5, 4, 8), mk(2, 7, 2, 8), mk(2, 7, 2, 8), mk(2, 5, 4, 8)
    lens = torch.tensor([7, 3])
    out, _ = ref.attention(q, k, v, lens, True, do=do)
    x = [q, k, v]
    for i in range(3):
        d = mk(*x[i].shape)
        h = 2.0 ** -10
        f = []
        for s in (1, -1):
            y = list(x)
            y[i] = x[i] + s * h * d                          # exact enough in fp32: the formula sees what it was given
            step = y[i].double() - x[i].double()
            f.append(((ref.attention(*y, lens, True)[0][0] * do.double()).sum(), (out[1 + i] * step).sum()))
        assert abs((f[0][0] - f[1][0]) - (f[0][1] - f[1][1])) < 1e-6 * out[1 + i].numel()
    xx, dy, gm, bt = mk(6, 9), mk(6, 9), mk(9), mk(9)
    out, _ = ref.frame_norm(xx, gm, bt, 1e-6, dy)
    leaves = [t.double().requires_grad_(True) for t in (xx, gm, bt)]
    y = torch.nn.functional.layer_norm(leaves[0], (9,), leaves[1], leaves[2], 1e-6)
    for a, b in zip(out[1:], torch.autograd.grad(y, leaves, dy.double())):
        assert torch.allclose(a, b, rtol=1e-9, atol=1e-11)


def test_dual_path_attention_model_config_and_keys(tmp_path):
    from dprnn_cases import SMALL
    from speech_amd.models.dprnn_tasnet import DPRNNTasNet
    cfg = dict(SMALL, sep_hidden_channels=32, rnn_type='attention', sep_num_heads=2)
    m = DPRNNTasNet(**cfg)
    unit = m.separator.dprnn.net[0].inter_chunk_block
    assert unit.attention.num_heads == 2 and unit.attention.causal is False
    assert DPRNNTasNet(**dict(cfg, causal=True)).separator.dprnn.net[0].inter_chunk_block.attention.causal is True
    assert DPRNNTasNet(**dict(cfg, causal=True)).separator.dprnn.net[0].intra_chunk_block.attention.causal is False
    assert sorted(k for k in unit.state_dict()) == ["attention.in_proj.bias", "attention.in_proj.weight", "fc.bias", "fc.weight",
                                                    "norm1d.bias", "norm1d.weight"]
    path = str(tmp_path / "m.pth")
    torch.save(dict(m.get_config(), state_dict=m.state_dict()), path)
    b = DPRNNTasNet.build_model(path, load_state_dict=True)
    assert b.get_config() == m.get_config() and b.sep_num_heads == 2
    assert all(torch.equal(x, y) for x, y in zip(m.state_dict().values(), b.state_dict().values()))
    assert "sep_num_heads" not in DPRNNTasNet(**SMALL).get_config()
    with pytest.raises(NotImplementedError, match="Not support gru"):
        DPRNNTasNet(**dict(SMALL, rnn_type='gru'))


@pytest.mark.parametrize("hidden,heads", [(32, 0), (32, -1), (32, 3), (24, 2), (288, 2)])
def test_self_attention_refuses_head_counts(hidden, heads):
    from dprnn_cases import SMALL
    from speech_amd.models.dprnn_tasnet import DPRNNTasNet
    from speech_amd.modules.attention import SelfAttention
    with pytest.raises(ValueError, match="num_heads times a multiple of 8"):
        SelfAttention(16, hidden, num_heads=heads)
    with pytest.raises(ValueError, match="num_heads times a multiple of 8"):
        DPRNNTasNet(**dict(SMALL, sep_hidden_channels=hidden, rnn_type='attention', sep_num_heads=heads))


def test_attention_workspace_of_every_size_the_wrapper_asks_for():
    for code in (_lib.TYPE_F32, _lib.TYPE_BF16):
        assert ops._attn_ws(2, 300, 300, 2, 1, 16, code, False, True) >= 2 * 2 * 300
        assert ops._attn_ws(2, 3, 3, 2, 1, 40, code, False, True) >= 2 * 2 * 3
        assert ops._attn_ws(2, 300, 300, 2, 1, 16, code, True, False) == 0
        assert ops._attn_ws(1, 1, 100000, 2, 1, 16, code, False, False) > 0
    with pytest.raises(_lib.CtnError):
        ops._attn_ws(2, 3, 3, 2, 1, 12, _lib.TYPE_F32, False, True)
