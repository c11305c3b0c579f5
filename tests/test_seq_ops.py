"""CPU: what the sequence operators (layer_norm, gru_scan, gated_mlp) refuse, at the C boundary and in Python, and the sizes of their workspaces."""
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from motif_amd.csrc import build
    build.build()
    from motif_amd import _lib
    return _lib.load()


@pytest.fixture(scope="module")
def ops(lib):
    from motif_amd import ops
    return ops


EINVAL, ELIMIT = -1, -2
P = 4096                                                 # an address that no refused call follows


def test_layer_norm_refuses_bad_arguments_before_it_launches(lib):
    fwd = lambda x=P, rs=8, y=P, rows=4, d=8, dt=0, pdt=0: lib.motif_layer_norm_fwd(x, rs, None, None, y, None, rows, d, 1e-5, dt, pdt, None)  # noqa: E731
    assert fwd(x=None) == fwd(y=None) == fwd(rows=-1) == fwd(d=0) == fwd(dt=3) == fwd(pdt=-1) == fwd(rs=-8) == EINVAL
    assert fwd(d=16385) == fwd(rows=1 << 31) == ELIMIT
    assert fwd(x=None, y=None, rows=0) == 0              # nothing to do
    bwd = lambda x=P, dy=P, st=P, dx=P, dw=None, ws=None, rows=4, d=8, dt=0: lib.motif_layer_norm_bwd(x, 8, dy, 8, None, st, dx, dw, None, ws, rows, d, dt, 0, None)  # noqa: E731
    assert bwd(x=None) == bwd(dy=None) == bwd(st=None) == bwd(dx=None) == bwd(dw=P) == bwd(rows=0) == bwd(dt=7) == EINVAL
    assert bwd(d=20000) == ELIMIT
    assert lib.motif_layer_norm_bwd_ws_floats(0, 5) == 0 and lib.motif_layer_norm_bwd_ws_floats(3, 0) == EINVAL and lib.motif_layer_norm_bwd_ws_floats(1, 16385) == ELIMIT
    for rows, d in ((1, 1), (10 ** 9, 64), (10 ** 6, 16384)):      # bounded: a share of the rows per workgroup
        assert 2 * d <= lib.motif_layer_norm_bwd_ws_floats(rows, d) <= 1024 * 2 * d


def test_gru_scan_refuses_bad_arguments_before_it_launches(lib):
    def fwd(z=P, q=P, h=P, cu=None, S=0, ws=P, B=2, T=4, D=8, dt=0, rs=8):
        return lib.motif_gru_scan_fwd(z, 32, rs, q, 32, rs, None, cu, S, h, P, ws, B, T, D, dt, None)
    assert fwd(z=None) == fwd(q=None) == fwd(h=None) == fwd(B=0) == fwd(T=-1) == fwd(T=0) == fwd(D=0) == fwd(dt=4) == fwd(rs=-8) == EINVAL
    assert fwd(cu=P, S=0, B=1) == fwd(cu=P, S=3, B=2) == EINVAL
    assert fwd(cu=P, S=3, B=1, ws=None) == fwd(B=1, T=100000, ws=None) == EINVAL        # a workspace is needed
    assert fwd(D=1 << 28) == fwd(T=1 << 31) == fwd(B=1 << 29) == ELIMIT
    assert fwd(B=1, T=100000, rs=(1 << 22) + 1) == ELIMIT
    bwd = lambda h=P, dh=P, dz=P, T=4: lib.motif_gru_scan_bwd(P, 32, 8, P, 32, 8, None, None, 0, h, dh, 32, 8, None, dz, None, None, P, 2, T, 8, 0, None)  # noqa: E731
    assert bwd(h=None) == bwd(dh=None) == bwd(dz=None) == bwd(T=0) == EINVAL
    ws = lib.motif_gru_scan_ws_floats
    assert ws(3, 16, 1 << 20, 0, 0) == 0 and ws(1, 1, 5, 0, 1) == 0
    assert ws(1, 7, 100, 1, 2) >= 7 and ws(1, 65536, 1024, 0, 1) > 0
    assert ws(0, 4, 4, 0, 0) == EINVAL and ws(1, 4, 1 << 28, 0, 0) == ELIMIT


def test_gated_mlp_refuses_bad_arguments_before_it_launches(lib):
    def fwd(x=P, wg=P, wu=P, h=P, G=None, U=None, ws=P, M=100, K=64, F=64, act=1, dt=1, rs=64):
        return lib.motif_gated_mlp_fwd(x, rs, wg, wu, None, None, h, G, U, ws, M, K, F, act, dt, None)
    assert fwd(x=None) == fwd(wg=None) == fwd(wu=None) == fwd(h=None) == fwd(M=-1) == fwd(K=0) == fwd(F=0) == fwd(act=3) == fwd(act=-1) == fwd(dt=5) == fwd(rs=-1) == EINVAL
    assert fwd(G=P) == fwd(U=P) == EINVAL                # both or neither
    assert fwd(M=5000, F=1024, dt=0, K=128, rs=128, ws=None) == fwd(M=5000, F=1024, K=65, rs=65, ws=None) == EINVAL      # operands to be laid out need a workspace
    assert fwd(K=65537) == fwd(F=65537) == fwd(M=(1 << 22) + 1) == ELIMIT
    assert fwd(x=None, M=0) == 0
    def bwd(G=P, dh=P, dx=P, dwg=P, dwu=P, ws=P, M=100):
        return lib.motif_gated_mlp_bwd(P, 64, P, P, G, P, dh, 64, dx, dwg, dwu, None, None, ws, M, 64, 64, 1, 1, None)
    assert bwd(G=None) == bwd(dh=None) == bwd(dwg=None) == bwd(dwu=None) == bwd(ws=None) == bwd(M=0) == bwd(dx=None, dwg=None, dwu=None) == bwd(G=P + 4) == EINVAL
    ws = lib.motif_gated_mlp_ws_bytes
    assert ws(P, 64, P, P, 64, 64, 64, 0) == 0           # few rows: none
    assert ws(P, 128, P, P, 5000, 128, 1024, 0) >= 3 * 2 * (5000 + 2048) * 128
    assert ws(P, 128, P, P, 100, 128, 64, 0) == 0         # small products: none
    assert ws(P, 64, P, P, 65, 64, 64, 0) == 0           # narrow layers: none
    assert ws(P, 64, P, P, 100, 70000, 64, 1) == ELIMIT


def test_python_refuses_shapes_types_and_host_tensors(ops):
    x = torch.zeros(4, 8)
    for call, match in ((lambda: ops.layer_norm(x.double()), "fp32, bf16 or fp16"), (lambda: ops.layer_norm(torch.zeros(())), "last axis"),
                        (lambda: ops.layer_norm(torch.zeros(2, 0)), "last axis"), (lambda: ops.layer_norm(torch.zeros(1, 16385)), "last axis"),
                        (lambda: ops.layer_norm(x, torch.ones(7)), "weight must be"), (lambda: ops.layer_norm(x, torch.ones(8).half()), "weight must be"),
                        (lambda: ops.layer_norm(x.half(), torch.ones(8), torch.ones(8).half()), "bias must be"), (lambda: ops.layer_norm(x), "CUDA")):
        with pytest.raises(RuntimeError, match=match):
            call()
    z = torch.zeros(2, 3, 8)
    cu = torch.zeros(3, dtype=torch.int32)
    for call, match in ((lambda: ops.gru_scan(x, x), "q must be"), (lambda: ops.gru_scan(z, z, cu_seqlens=cu), "q must be"), (lambda: ops.gru_scan(z[:1], z), "z must be"),
                        (lambda: ops.gru_scan(z.half(), z), "z must be"), (lambda: ops.gru_scan(z, z, torch.zeros(3, 8)), "h0 must be"),
                        (lambda: ops.gru_scan(z, z, torch.zeros(2, 8).half()), "h0 must be"), (lambda: ops.gru_scan(x, x, cu_seqlens=cu.long()), "cu_seqlens"),
                        (lambda: ops.gru_scan(x, x, cu_seqlens=cu[:1]), "cu_seqlens"), (lambda: ops.gru_scan(x, x, torch.zeros(3, 8), cu), "h0 must be"),
                        (lambda: ops.gru_scan(z.int(), z.int()), "fp32, bf16 or fp16"), (lambda: ops.gru_scan(z, z), "CUDA")):
        with pytest.raises(RuntimeError, match=match):
            call()
    w = torch.zeros(5, 8)
    for call, match in ((lambda: ops.gated_mlp(x, w, w, act="relu"), "act must be"), (lambda: ops.gated_mlp(x, w[:, :7], w), "K"), (lambda: ops.gated_mlp(x, w, w[:4]), "w_up must be"),
                        (lambda: ops.gated_mlp(x, w.half(), w.half()), "w_gate must be"), (lambda: ops.gated_mlp(x, w, w, torch.zeros(4)), "b_gate must be"),
                        (lambda: ops.gated_mlp(x, w, w, None, torch.zeros(5).half()), "b_up must be"), (lambda: ops.gated_mlp(x.double(), w, w), "fp32, bf16 or fp16"),
                        (lambda: ops.gated_mlp(x, torch.zeros(0, 8), torch.zeros(0, 8)), "K"), (lambda: ops.gated_mlp(x, w, w), "CUDA")):
        with pytest.raises(RuntimeError, match=match):
            call()


def test_the_modules_hold_torchs_parameters(ops):
    from motif_amd.models.modules.layers import GatedMLP, LayerNorm
    n, m = LayerNorm(24), GatedMLP(24, 40)
    assert {k: tuple(v.shape) for k, v in n.state_dict().items()} == {"weight": (24,), "bias": (24,)}
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {"gate.weight": (40, 24), "gate.bias": (40,), "up.weight": (40, 24), "up.bias": (40,)}
    n.load_state_dict(torch.nn.LayerNorm(24).state_dict())
    for module in (n, m):
        with pytest.raises(RuntimeError, match="CUDA"):
            module(torch.zeros(2, 24))


def test_forward_mode_is_refused_wherever_a_tangent_comes_in(ops):
    """An output without a tangent counts as one whose derivative is zero: a silent wrong answer."""
    from torch.autograd import forward_ad
    calls = ((lambda x, w, b: ops.layer_norm(x, w, b), ((4, 8), (8,), (8,))),
             (lambda z, q, h0: ops.gru_scan(z, q, h0), ((2, 3, 8), (2, 3, 8), (2, 8))),
             (lambda x, wg, wu, bg, bu: ops.gated_mlp(x, wg, wu, bg, bu), ((4, 8), (5, 8), (5, 8), (5,), (5,))))
    for call, shapes in calls:
        tensors = [torch.zeros(s) for s in shapes]
        for i in range(len(tensors)):
            with forward_ad.dual_level():
                duals = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(tensors)]
                for mode in (torch.enable_grad, torch.no_grad):
                    with mode(), pytest.raises(RuntimeError, match="forward-mode"):
                        call(*duals)
                with pytest.raises(RuntimeError, match="CUDA"):          # no tangent: as outside
                    call(*tensors)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(call, tuple(tensors), tuple(torch.ones_like(t) for t in tensors))
        with pytest.raises(RuntimeError, match="CUDA"):
            call(*tensors)


def test_gru_scan_gives_time_slots_to_few_channels_whatever_their_number_of_batches(lib):
    """Long sequences are walked by one lane per channel only where channels are many; a workspace (of segments) means time slots.  What a grid cannot hold is
    refused."""
    ws = lib.motif_gru_scan_ws_floats
    for B in (1, 100, 511, 512):                          # (beyond, one segment to a batch fills the chip)
        assert ws(B, 8192, 16, 0, 1) > 0, B
    assert ws(512, 65536, 1024, 0, 1) == 0 and ws(1, 4096, 1 << 20, 0, 0) == 0
    fwd = lambda B, T, D: lib.motif_gru_scan_fwd(P, T * D, D, P, T * D, D, None, None, 0, P, P, P, B, T, D, 0, None)  # noqa: E731
    assert fwd(1 << 25, 1, 1024) == fwd((1 << 29) - 1, 2, 40) == ELIMIT
