"""What rms_norm, linear and the AdamW step refuse, without a GPU: checks of arguments come before any launch."""
import ctypes as C

import pytest
import torch

from selfc_amd import _lib, optim, pointwise as pw


def f(*s, dt=torch.float16):
    return torch.zeros(*s, dtype=dt)


@pytest.fixture
def on_cpu(monkeypatch):
    """the checks behind the device's: shapes and types of CPU tensors, with every launch turned into an error"""
    monkeypatch.setattr(_lib, "require_gpu", lambda t: None)
    monkeypatch.setattr(_lib, "host", lambda: pytest.fail("launched"))


def test_cpu_tensors_are_refused():
    for call in (lambda: pw.rms_norm(f(2, 4), f(4)), lambda: pw.rms_norm_q8(f(2, 4), f(4)), lambda: pw.linear(f(2, 4), f(3, 4)),
                 lambda: pw.linear_q8(f(2, 4).to(torch.float8_e4m3fn), f(2, dt=torch.float32), f(3, 4).to(torch.float8_e4m3fn), f(3, dt=torch.float32)),
                 lambda: optim.grad_norm([f(3)]), lambda: optim.adamw_step([f(3)], [f(3)], f(256, dt=torch.float32), f(256, dt=torch.float32), step=1, lr=1e-3)):
        with pytest.raises(RuntimeError, match="MI355X"):
            call()


@pytest.mark.parametrize("call,what", [
    (lambda: pw.rms_norm(f(2, 4, dt=torch.float64), f(4, dt=torch.float64)), "float64"),
    (lambda: pw.rms_norm(f(2, 4), f(4, dt=torch.bfloat16)), "weight"),
    (lambda: pw.rms_norm(f(2, 4), f(5)), "weight"),
    (lambda: pw.rms_norm(f(2, 4), f(4), residual=f(3, 4)), "residual"),
    (lambda: pw.rms_norm(f(2, 4), f(4), residual=f(2, 4, dt=torch.bfloat16)), "residual"),
    (lambda: pw.rms_norm(f(1, 16385), f(16385)), "16384"),
    (lambda: pw.rms_norm(f(2, 0), f(0)), "rows of"),
    (lambda: pw.rms_norm(f(2, 4), f(4), eps=-1.0), "eps"),
    (lambda: pw.linear(f(2, 4), f(3, 5)), "weight"),
    (lambda: pw.linear(f(2, 4), f(3, 4, dt=torch.bfloat16)), "weight"),
    (lambda: pw.linear(f(2, 4, dt=torch.float32), f(3, 4, dt=torch.float32)), "float32"),
    (lambda: pw.linear(f(2, 4), f(3, 4), bias=f(4)), "bias"),
    (lambda: pw.linear(f(2, 4), f(3, 4), residual=f(2, 4)), "residual"),
    (lambda: pw.linear(f(2, 4), f(3, 4), act="tanh"), "act"),
    (lambda: pw.linear(f(2, 0), f(3, 0)), "weight"),
])
def test_shapes_and_types_are_checked(on_cpu, call, what):
    with pytest.raises(RuntimeError, match=what):
        call()


def test_q8_forms_have_no_gradient(on_cpu):
    w = torch.zeros(4, dtype=torch.float16, requires_grad=True)
    with pytest.raises(NotImplementedError):
        pw.rms_norm_q8(f(2, 4), w)
    e = torch.float8_e4m3fn
    with pytest.raises(NotImplementedError):
        pw.linear_q8(f(2, 4).to(e), f(2, dt=torch.float32), f(4, 4).to(e), f(4, dt=torch.float32), bias=w, out_dtype=torch.float16)
    with pytest.raises(RuntimeError, match="x_scale"):
        pw.linear_q8(f(2, 4).to(e), f(3, dt=torch.float32), f(4, 4).to(e), f(4, dt=torch.float32))
    with pytest.raises(RuntimeError, match="out_dtype"):
        pw.linear_q8(f(2, 4).to(e), f(2, dt=torch.float32), f(4, 4).to(e), f(4, dt=torch.float32), out_dtype=torch.float64)


def test_quantize_rows():
    w = torch.randn(5, 40)
    w[2] = 0
    q, s = pw.quantize_rows(w)
    assert q.dtype == torch.float8_e4m3fn and s[2] == 1 and not q[2].float().any()
    assert ((q.float() * s[:, None] - w).abs() <= w.abs() * 2.0 ** -4 * 1.001 + s[:, None] * 2.0 ** -10).all()


def test_adamw_step_checks(monkeypatch):
    monkeypatch.setattr(_lib, "require_gpu", lambda t: None)
    monkeypatch.setattr(optim.rt, "call", lambda *a: pytest.fail("launched"))
    m = lambda n, dt=torch.float32: torch.zeros(n, dtype=dt)  # noqa: E731
    ok = dict(step=1, lr=1e-3)
    with pytest.raises(RuntimeError, match="gradient 0"):
        optim.adamw_step([m(3)], [m(4)], m(256), m(256), **ok)
    with pytest.raises(RuntimeError, match="tensor 1"):
        optim.adamw_step([m(3), m(3, torch.float16)], [m(3), m(3, torch.float16)], m(512), m(512), **ok)
    with pytest.raises(RuntimeError, match="exp_avg"):
        optim.adamw_step([m(257)], [m(257)], m(256), m(512), **ok)
    with pytest.raises(RuntimeError, match="scales"):
        optim.adamw_step([m(3)], [m(3)], m(256, torch.float8_e4m3fn), m(256, torch.float8_e5m2), **ok)
    with pytest.raises(RuntimeError, match="moments"):
        optim.adamw_step([m(3)], [m(3)], m(256, torch.float16), m(256), **ok)
    with pytest.raises(RuntimeError, match="step"):
        optim.adamw_step([m(3)], [m(3)], m(256), m(256), step=0, lr=1e-3)
    with pytest.raises(RuntimeError, match="stretch"):
        t = torch.zeros(4, 6)[:, :3]
        optim.adamw_step([t], [t], m(256), m(256), **ok)
    with pytest.raises(RuntimeError, match="betas"):
        optim.adamw_step([m(3)], [m(3)], m(256), m(256), beta1=1.0, **ok)
    optim.adamw_step([], [], m(0), m(0), **ok)
    t, big = m(3), m(600)
    for twice in ([t, t], [big[:300], big[299:]], [big, m(2), big[5:6]]):
        with pytest.raises(RuntimeError, match="share memory"):
            optim.adamw_step(twice, [x.clone() for x in twice], m(2048), m(2048), **ok)
    with pytest.raises(RuntimeError, match="same memory"):
        optim.adamw_step([t], [m(3)], big, big, **ok)


def test_c_entries_refuse_without_launching():
    L = _lib.lib()
    one = C.c_void_p(16)          # never read: every call below is refused by its arguments
    assert L.selfc_rmsnorm(None, 4, None, 4, one, 1, None, one, None, 2, 4, 2, 1e-6, None) == -1
    assert L.selfc_rmsnorm(one, 4, one, 4, one, 1, None, one, None, 2, 4, 2, 1e-6, None) == -1           # a residual without its sum
    assert L.selfc_rmsnorm(one, 4, None, 4, one, 1, None, one, None, 2, 16385, 2, 1e-6, None) == -1
    assert L.selfc_rmsnorm(one, 4, None, 4, one, 1, None, one, None, 0, 4, 2, 1e-6, None) == 0           # no rows
    assert L.selfc_linear(C.c_void_p(8), 8, one, 8, None, None, None, 0, None, 0, one, None, None, 32, 8, 8, 2, 2, None) == -1   # not aligned
    assert L.selfc_linear(one, 9, one, 8, None, None, None, 0, None, 0, one, None, None, 32, 8, 8, 2, 2, None) == -1             # pitch
    assert L.selfc_linear(one, 8, one, 8, None, None, None, 7, None, 0, one, None, None, 2, 8, 8, 2, 2, None) == -1             # activation
    assert L.selfc_linear(one, 16, one, 16, None, None, None, 0, None, 0, one, None, None, 2, 8, 16, 3, 2, None) == -1          # scales missing
    assert L.selfc_linear(one, 8192, one, 8192, None, None, None, 0, None, 0, one, None, None, 64, 64, 8192, 2, 2, None) == -1  # workspace missing
    assert L.selfc_linear_ws_floats(64, 64, 8192, 2) > 0 and L.selfc_linear_ws_floats(0, 64, 64, 2) == 0
    assert L.selfc_linear_dw(one, 8, one, 8, one, None, None, 0, 8, 8, 2, None) == -1
    assert L.selfc_pack_rows(one, 5, one, 2, 5, 7, 2, None) == -1
    assert L.selfc_linear(one, 7, one, 7, None, None, None, 0, None, 0, one, None, None, 2, 8, 7, 2, 2, None) == -1              # below one piece
    assert L.selfc_linear(C.c_void_p(17), 9, one, 9, None, None, None, 0, None, 0, one, None, None, 2, 8, 9, 2, 2, None) == -1   # half a value off
    assert [L.selfc_linear_any_layout(r, k, e) for r, k, e in ((16, 8, 2), (17, 8, 2), (1, 7, 2), (1, 16, 1), (1, 15, 1), (1, 9000, 2))] == [1, 0, 0, 1, 0, 0]
    assert L.selfc_linear_dz(one, 8, one, 9, one, 8, None, None, 2, 8, 2, None) == -1                    # activation
    assert L.selfc_linear_dz(one, 8, C.c_void_p(8), 3, one, 8, None, None, 2, 8, 2, None) == -1          # 16-bit codes, not aligned
    assert L.selfc_linear_rows_bwd(one, 8, one, 9, one, 8, one, None, 2, 8, 8, 2, None) == -1            # activation
    assert L.selfc_linear_rows(one, 8, one, 8, None, 4, None, 0, one, C.c_void_p(8), None, 2, 8, 8, 2, None) == -1
    assert L.selfc_pack_rows(None, 5, None, 0, 5, 8, 2, None) == 0                                       # no rows: no memory either
    assert L.selfc_adamw_block() == optim.BLOCK


def test_nets_in_the_dense_blocks_layout_refuse_ffnet():
    from selfc_amd.modules import SelfC_GMM_arch_inv as big
    from selfc_amd.modules.Subnet_constructor import FFNet, subnet
    with pytest.raises(NotImplementedError, match="FFNet"):
        big.SelfCInvNet({"global_module": "nonlocal", "stp_blk_num": 2, "fh_loss": "l2", "scale": 4, "gmm_k": 5}, 3, 3, "FFNet", [1, 1], 2)
    net = subnet("FFNet", "xavier")(9, 3)
    assert isinstance(net, FFNet) and net.width == 64 and not net.out.weight.any()
    with pytest.raises(NotImplementedError):
        FFNet(3, 3, width=20)


@pytest.mark.parametrize("needs_grad", [False, True])
def test_tangents_are_refused(monkeypatch, needs_grad):
    """An input of forward-mode derivatives would lose them; the check comes before the first launch."""
    import torch.autograd.forward_ad as fw
    h = _lib.host()
    x, w, b, r, n, one = f(2, 4), f(3, 4), f(3), f(2, 3), f(4), torch.ones(2)
    e = torch.float8_e4m3fn
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t.requires_grad_(needs_grad), torch.ones_like(t))  # noqa: E731
        calls = [lambda: h.linear(dual(x), w, b, r, 0, needs_grad, 0), lambda: h.linear(x, dual(w), None, None, 0, needs_grad, 0),
                 lambda: h.linear(x, w, dual(b), None, 0, needs_grad, 0), lambda: h.linear(x, w, None, dual(r), 0, needs_grad, 0),
                 lambda: h.norm(dual(x), None, n, 1e-6, False, needs_grad, 0), lambda: h.norm(x, dual(f(2, 4)), n, 1e-6, False, needs_grad, 0),
                 lambda: h.norm(x, None, dual(n), 1e-6, not needs_grad, needs_grad, 0),
                 lambda: h.linear_q8(x.detach().to(e), dual(one), w.detach().to(e), torch.ones(3), None, None, 0, 2, 0)]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


@pytest.mark.parametrize("capturable", [False, True])
def test_a_refused_step_leaves_everything_as_it_was(monkeypatch, capturable):
    """A group whose gradients are refused: no group's step is counted and nothing is launched; afterwards the count goes on from there."""
    launched = []
    monkeypatch.setattr(_lib, "require_gpu", lambda t: None)
    monkeypatch.setattr(optim, "on_device", lambda t: optim.torch.no_grad())
    monkeypatch.setattr(optim, "_stream", lambda t: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(optim.rt, "call", lambda *a: launched.append(a))
    ps = [torch.nn.Parameter(torch.zeros(n, 3)) for n in (4, 300, 2)]
    opt = optim.AdamW([{"params": ps[:1]}, {"params": ps[1:]}], capturable=capturable)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    assert len(launched) == 2
    good, ps[2].grad = ps[2].grad, torch.ones(2, 3).to_sparse()
    for _ in range(3):
        with pytest.raises(RuntimeError, match="gradient 1"):
            opt.step()
    assert len(launched) == 2 and all(opt.state[p]["step"].item() == 1 for p in ps)
    ps[2].grad = good
    opt.step()
    assert len(launched) == 4 and all(opt.state[p]["step"].item() == 2 for p in ps)
    if not capturable:
        assert [a[15] for a in launched] == [1, 1, 2, 2]               # the numbers that the launches got


def test_moments_that_overlap_are_refused(monkeypatch):
    monkeypatch.setattr(_lib, "require_gpu", lambda t: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    buf, launched = torch.zeros(2048), []
    monkeypatch.setattr(optim, "on_device", lambda t: optim.torch.no_grad())
    monkeypatch.setattr(optim, "_stream", lambda t: 0)
    monkeypatch.setattr(optim.rt, "call", lambda *a: launched.append(a))
    p, ok = [torch.zeros(300)], dict(step=1, lr=1e-3)
    for m, v in ((buf, buf[511:]), (buf[256:], buf), (buf, buf[:512])):
        with pytest.raises(RuntimeError, match="memory"):
            optim.adamw_step(p, [torch.ones(300)], m, v, **ok)
    codes, s = torch.zeros(2048, dtype=torch.uint8), torch.ones(8)
    m8, v8 = codes.view(torch.float8_e4m3fn), codes.view(torch.float8_e5m2)
    for args in ((m8, v8[511:], s[:2], s[2:]), (m8, v8[512:], s, s[1:]), (m8, v8[512:], s, s), (m8, v8[512:], codes[1020:1028].view(torch.float32), s)):
        with pytest.raises(RuntimeError, match="memory"):
            optim.adamw_step(p, [torch.ones(300)], *args, **ok)
    assert not launched
    optim.adamw_step(p, [torch.ones(300)], buf, buf[512:], **ok)                 # the step uses 512 values of each
    optim.adamw_step(p, [torch.ones(300)], m8, v8[512:], s, s[2:], **ok)
    assert len(launched) == 2


@pytest.mark.parametrize("cols,lanes", [(1, 8), (64, 8), (65, 16), (256, 32), (257, 64), (2048, 64), (2049, 256), (16384, 256)])
def test_more_lanes_than_a_launch_has_are_refused(cols, lanes):
    """Counts of rows that need 2^32 lanes: refused before a launch (whose size would not fit)."""
    L, one = _lib.lib(), C.c_void_p(16)          # never read: refused by their numbers
    for rows in (2 ** 32 // lanes, 2 ** 31 - 1, 2 ** 40):
        assert L.selfc_rmsnorm(one, cols, None, 0, one, 1, None, one, None, rows, cols, 2, 1e-6, None) == -1
        assert L.selfc_rmsnorm_bwd(one, cols, one, 1, one, None, one, None, None, rows, cols, 2, 1e-6, None) == -1
    assert L.selfc_pack_rows(one, 5, one, 2 ** 32, 5, 8, 2, None) == -1
    assert L.selfc_pack_rows(one, 20, one, 2 ** 31, 20, 32, 1, None) == -1
