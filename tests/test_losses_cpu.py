"""CPU: what the linear cross entropy and the clipping refuse, before any launch (no GPU needed)."""
import ctypes

import pytest
import torch


def test_losses_refuse_bad_arguments():
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = torch.zeros(4, 16), torch.zeros(10, 16), torch.zeros(4, dtype=torch.int64)
    for bad in (lambda: linear_cross_entropy(h, w, t),                                  # not on a CUDA device
                lambda: linear_cross_entropy(h, w, t, reduction="average"),
                lambda: linear_cross_entropy(h.half(), w.half(), t),
                lambda: linear_cross_entropy(h.bfloat16(), w, t),
                lambda: linear_cross_entropy(h, w, t.float())):
        with pytest.raises(ValueError):
            bad()


def test_sizes_the_kernels_do_not_take():
    from hffn_b200 import _native as n
    from hffn_b200.losses import _sizes
    assert min(_sizes(n.F32, 100, 64, 1000)) > 0
    for n_tokens, d, vocab in ((100, 32776, 1000), (1 << 24, 64, 1 << 24), (100, 64, (1 << 24) + 1)):
        with pytest.raises(ValueError):
            _sizes(n.BF16, n_tokens, d, vocab)


def test_linear_ce_entries_refuse_bad_arguments():
    from hffn_b200 import _native as n
    lib = n.lib
    state, work = lib.hffn_linear_ce_state_bytes, lib.hffn_linear_ce_backward_workspace
    assert state(n.F32, 46, 128, 1024) >= 256 * 128 * 4 and work(n.BF16, 46, 128, 1024) > 0
    for bad in ((7, 4, 16, 10), (n.F32, 0, 16, 10), (n.F32, (1 << 24) + 1, 16, 10), (n.F32, 4, 12, 10),
                (n.F32, 4, 0, 10), (n.F32, 4, 16, 0)):
        assert state(*bad) == -1 and work(*bad) == -1 and lib.hffn_linear_ce_forward_workspace(*bad) == -1

    def forward(dtype=n.F32, hidden=16, stride=16, weight=16, targets=16, reduction=0, loss=16, buffer=16, rows=4, d=16,
                vocab=10):
        return lib.hffn_linear_ce_forward(dtype, hidden, stride, weight, targets, -100, reduction, 1, loss, buffer, buffer,
                                          rows, d, vocab, None)

    for bad in (dict(dtype=5), dict(hidden=None), dict(weight=None), dict(targets=None), dict(loss=None),
                dict(buffer=None), dict(reduction=3), dict(rows=0), dict(d=20), dict(vocab=0), dict(stride=8),
                dict(weight=24), dict(buffer=8)):
        assert forward(**bad) == n.HFFN_ERR_ARGUMENT, bad
    assert b"16-byte" in lib.hffn_last_error()

    def backward(weight=16, reduction=0, upstream=16, hidden=16, grad=16, buffer=16, rows=4):
        return lib.hffn_linear_ce_backward(n.F32, weight, reduction, upstream, hidden, grad, buffer, buffer, rows, 16, 10,
                                           None)

    for bad in (dict(weight=None), dict(upstream=None), dict(buffer=None), dict(reduction=-1), dict(rows=-3),
                dict(hidden=8), dict(grad=4)):
        assert backward(**bad) == n.HFFN_ERR_ARGUMENT, bad


def test_clip_entries_refuse_bad_arguments():
    from hffn_b200 import _native as n
    lib = n.lib

    def call(ins=(256, 4096), outs=(256, 4096), counts=(10, 10), types=(0, 0), out_types=(0, 0), limit=1.0, norm=64,
             work=64):
        k = len(ins)
        return lib.hffn_clip_grad_norm(k, (ctypes.c_void_p * k)(*ins), (ctypes.c_void_p * k)(*outs),
                                       (ctypes.c_int64 * k)(*counts), (ctypes.c_int32 * k)(*types),
                                       (ctypes.c_int32 * k)(*out_types), limit, norm, work, None)

    for bad in (dict(limit=-1.0), dict(limit=float("nan")), dict(norm=None), dict(work=None), dict(work=12),
                dict(types=(0, 2)), dict(out_types=(9, 0)), dict(counts=(10, -1)), dict(counts=(1 << 40, 1)),
                dict(ins=(256, None)), dict(outs=(None, 4096)), dict(ins=(258, 4096)), dict(outs=(256, 4097)),
                dict(outs=(256, 256)), dict(outs=(256, 280)), dict(outs=(4096, 256)), dict(outs=(260, 4096)),
                dict(ins=(256, 256)), dict(outs=(256, 4096), out_types=(1, 0))):
        assert call(**bad) == n.HFFN_ERR_ARGUMENT, bad
    assert lib.hffn_grad_norm(-1, None, None, None, 64, 64, None) == n.HFFN_ERR_ARGUMENT
    assert lib.hffn_grad_norm(1, None, None, None, 64, 64, None) == n.HFFN_ERR_ARGUMENT
    assert lib.hffn_grad_norm_workspace(-1) == -1 and lib.hffn_grad_norm_workspace(0) > 0


def test_clip_refuses_host_tensors():
    from hffn_b200.grad_clip import clip_grad_norm, grad_norm
    with pytest.raises(ValueError):
        grad_norm([torch.zeros(3)])
    with pytest.raises(ValueError):
        clip_grad_norm([torch.zeros(3)], 1.0)


def test_workspaces_follow_the_path_taken():
    """Statistics of the few-row kernel's blocks only for few rows; head parts only where the call makes them."""
    from hffn_b200 import _native as n
    lib = n.lib
    assert lib.hffn_linear_ce_forward_workspace(n.BF16, 1 << 20, 64, 1024) < 100 << 20
    assert lib.hffn_linear_ce_state_bytes(n.F32, 1, 2048, 50304) < 8 << 20
    assert lib.hffn_linear_ce_state_bytes(n.F32, 17, 2048, 50304) >= 4 * 2048 * 50304
    assert lib.hffn_linear_ce_backward_workspace(n.F32, 1, 2048, 50304) >= 4 * 2048 * 50304
