"""Argument checks of the embedding, layer norm, log-probability and loss entry
points, in Python and in C.  No GPU."""
import pytest
import torch


def test_python_refusals():
    import advanced_optimizers_b200 as A
    x, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    cpu = [lambda: A.embedding(ids, x), lambda: A.layer_norm(x), lambda: A.layer_norm(x, torch.ones(8), torch.ones(8)),
           lambda: A.token_logprobs(x, ids), lambda: A.policy_loss(x, x, x), lambda: A.preference_loss(x)]
    for call in cpu:
        with pytest.raises(NotImplementedError, match="CUDA device"):
            call()
    with pytest.raises(ValueError, match="matrix"):
        A.embedding(ids, x[0])
    with pytest.raises(NotImplementedError, match="int32 or int64"):
        A.embedding(x, x)
    with pytest.raises(NotImplementedError, match="int32 or int64"):
        A.token_logprobs(x, x[:, 0])
    with pytest.raises(ValueError, match=r"logits \[\.\.\., V\]"):
        A.token_logprobs(x, ids[:3])
    with pytest.raises(ValueError, match="at least one dimension"):
        A.layer_norm(x.sum())
    with pytest.raises(ValueError, match=r"\[sequences, tokens\]"):
        A.policy_loss(x[0], x[0], x[0])
    with pytest.raises(ValueError, match=r"\[sequences, tokens\]"):
        A.preference_loss(x[0])


def test_packed_structs_match_the_header():
    from advanced_optimizers_b200 import _lib as L
    from advanced_optimizers_b200 import embeddings, losses, norms
    lib = L.lib()
    for which, s in ((13, embeddings._FORWARD), (14, embeddings._GRAD), (15, norms._FORWARD), (16, norms._GRAD), (17, losses._LOGPROBS),
                     (18, losses._POLICY), (19, losses._PREFERENCE)):
        assert lib.advopt_sizeof(which) == s.size


OK = {
    "advopt_embedding": dict(y=4096, weight=4096, ids=4096, err=0, ldw=8, tokens=4, vocab=5, width=8, dtype=1, id_bytes=8, scale=1.0, pad=0),
    "advopt_embedding_grad": dict(dweight=4096, dy=4096, ids=4096, work=4096, tokens=4, vocab=5, width=8, padding=-1, dtype=1, id_bytes=8, scale=1.0, pad=0),
    "advopt_layer_norm": dict(y=4096, x=4096, weight=0, bias=0, stats=0, ldx=8, rows=4, cols=8, eps=1e-5, x_dtype=1, w_dtype=0, pad=0),
    "advopt_layer_norm_grad": dict(dx=4096, dweight=4096, dbias=4096, dy=4096, x=4096, weight=4096, stats=4096, work=4096, lddy=8, ldx=8, rows=4, cols=8,
                                   x_dtype=1, w_dtype=0),
    "advopt_token_logprobs": dict(out=4096, stats=0, logits=4096, tokens=4096, err=0, work=0, inner=4, ld_outer=0, ld_inner=8, rows=4, vocab=8, ignore=-100,
                                  dtype=1, token_bytes=8, temperature=1.0, pad=0),
    "advopt_policy_loss": dict(loss=4096, kl=4096, clipped=4096, slope=0, scale=4096, logprobs=4096, old=4096, ref=0, advantages=4096, mask=0, work=4096, ld_logprobs=8,
                               ld_old=8, ld_ref=0, ld_adv=-1, ld_mask=0, rows=4, cols=8, log_high=0.2, log_low=-0.2, clip_low=0.2, clip_high=0.2,
                               kl_weight=0.0, by_rows=0, dtype=0, pad=0),
    "advopt_preference_loss": dict(loss=4096, rewards=4096, slope=0, logprobs=4096, ref=0, mask=0, work=4096, ld_logprobs=8, ld_ref=0, ld_mask=0, pairs=2,
                                   cols=8, beta=0.1, smoothing=0.0, average=0, dtype=0),
}
NAN, BIG = float("nan"), 1 << 40
BAD = [
    ("advopt_embedding", dict(tokens=-1)), ("advopt_embedding", dict(tokens=BIG)), ("advopt_embedding", dict(vocab=BIG)), ("advopt_embedding", dict(width=BIG)),
    ("advopt_embedding", dict(ldw=7)), ("advopt_embedding", dict(id_bytes=2)), ("advopt_embedding", dict(dtype=2)), ("advopt_embedding", dict(y=0)),
    ("advopt_embedding", dict(weight=0)), ("advopt_embedding", dict(ids=0)),
    ("advopt_embedding_grad", dict(tokens=-1)), ("advopt_embedding_grad", dict(vocab=BIG)), ("advopt_embedding_grad", dict(width=-3)),
    ("advopt_embedding_grad", dict(dtype=3)), ("advopt_embedding_grad", dict(id_bytes=1)), ("advopt_embedding_grad", dict(dweight=0)),
    ("advopt_embedding_grad", dict(dweight=4100)), ("advopt_embedding_grad", dict(tokens=300, work=4104)), ("advopt_embedding_grad", dict(tokens=300, work=0)),
    ("advopt_embedding_grad", dict(dy=0)), ("advopt_embedding_grad", dict(tokens=(1 << 31) - 1, width=(1 << 31) - 1)),
    ("advopt_layer_norm", dict(rows=-1)), ("advopt_layer_norm", dict(cols=BIG)), ("advopt_layer_norm", dict(ldx=7)), ("advopt_layer_norm", dict(eps=-1.0)),
    ("advopt_layer_norm", dict(eps=NAN)), ("advopt_layer_norm", dict(x_dtype=2)), ("advopt_layer_norm", dict(w_dtype=5)), ("advopt_layer_norm", dict(x=0)),
    ("advopt_layer_norm", dict(y=0)), ("advopt_layer_norm", dict(stats=4100)),
    ("advopt_layer_norm_grad", dict(rows=-1)), ("advopt_layer_norm_grad", dict(lddy=7)), ("advopt_layer_norm_grad", dict(ldx=7)),
    ("advopt_layer_norm_grad", dict(x_dtype=2)), ("advopt_layer_norm_grad", dict(work=0)), ("advopt_layer_norm_grad", dict(work=4100)),
    ("advopt_layer_norm_grad", dict(stats=0)), ("advopt_layer_norm_grad", dict(dy=0)),
    ("advopt_token_logprobs", dict(rows=-1)), ("advopt_token_logprobs", dict(vocab=0)), ("advopt_token_logprobs", dict(vocab=BIG)),
    ("advopt_token_logprobs", dict(inner=0)), ("advopt_token_logprobs", dict(token_bytes=3)), ("advopt_token_logprobs", dict(temperature=0.0)),
    ("advopt_token_logprobs", dict(temperature=NAN)), ("advopt_token_logprobs", dict(temperature=float("inf"))), ("advopt_token_logprobs", dict(dtype=9)),
    ("advopt_token_logprobs", dict(out=0)), ("advopt_token_logprobs", dict(rows=200, vocab=50257)), ("advopt_token_logprobs", dict(rows=200, vocab=50257, work=4100)), ("advopt_token_logprobs", dict(logits=0)), ("advopt_token_logprobs", dict(stats=4100)),
    ("advopt_policy_loss", dict(rows=-1)), ("advopt_policy_loss", dict(rows=BIG)), ("advopt_policy_loss", dict(loss=0)), ("advopt_policy_loss", dict(kl=0)), ("advopt_policy_loss", dict(clipped=0)),
    ("advopt_policy_loss", dict(scale=0)), ("advopt_policy_loss", dict(work=0)), ("advopt_policy_loss", dict(work=4104)),
    ("advopt_policy_loss", dict(ld_old=7)), ("advopt_policy_loss", dict(ld_adv=7)), ("advopt_policy_loss", dict(mask=4096, ld_mask=7)),
    ("advopt_policy_loss", dict(ref=4096, ld_ref=7)), ("advopt_policy_loss", dict(clip_low=1.5)), ("advopt_policy_loss", dict(clip_high=NAN)),
    ("advopt_policy_loss", dict(kl_weight=float("inf"))), ("advopt_policy_loss", dict(dtype=2)), ("advopt_policy_loss", dict(advantages=0)),
    ("advopt_preference_loss", dict(pairs=0)), ("advopt_preference_loss", dict(pairs=BIG)), ("advopt_preference_loss", dict(cols=-1)),
    ("advopt_preference_loss", dict(loss=0)), ("advopt_preference_loss", dict(rewards=0)), ("advopt_preference_loss", dict(beta=NAN)),
    ("advopt_preference_loss", dict(smoothing=1.1)), ("advopt_preference_loss", dict(ld_logprobs=7)), ("advopt_preference_loss", dict(mask=4096, ld_mask=3)),
    ("advopt_preference_loss", dict(work=4100)), ("advopt_preference_loss", dict(dtype=4)),
]


@pytest.mark.parametrize("name,bad", BAD, ids=lambda v: v if isinstance(v, str) else "-".join(map(str, v)))
def test_c_entries_refuse_before_they_launch(name, bad):
    from advanced_optimizers_b200 import _lib as L
    from advanced_optimizers_b200 import embeddings, losses, norms
    packer = {"advopt_embedding": embeddings._FORWARD, "advopt_embedding_grad": embeddings._GRAD, "advopt_layer_norm": norms._FORWARD,
              "advopt_layer_norm_grad": norms._GRAD, "advopt_token_logprobs": losses._LOGPROBS, "advopt_policy_loss": losses._POLICY,
              "advopt_preference_loss": losses._PREFERENCE}[name]
    fields = {**OK[name], **bad}
    assert len(fields) == len(OK[name]), "a field that the call does not have"
    rc = getattr(L.lib(), name)(packer.pack(*fields.values()), None)
    assert rc in (-1, -3) and L.lib().advopt_last_error()
    assert getattr(L.lib(), name)(None, None) == -1


def test_gradient_entries_refuse_before_they_launch():
    from advanced_optimizers_b200 import _lib as L
    from advanced_optimizers_b200 import losses
    lib = L.lib()
    args = losses._LOGPROBS.pack(*{**OK["advopt_token_logprobs"], "stats": 4096}.values())
    for bad in ((0, 4096, args), (4104, 4096, args), (4096, 0, args), (4096, 4096, None), (4096, 4096, losses._LOGPROBS.pack(*OK["advopt_token_logprobs"].values()))):
        assert lib.advopt_token_logprobs_grad(*bad, None) == -1
    good = [4096, 4096, 4096, 4096, 4, 8, 0]
    for at, v in ((0, 0), (1, 0), (2, 0), (3, 0), (4, -1), (5, BIG), (6, 7)):
        assert lib.advopt_policy_loss_grad(*good[:at], v, *good[at + 1 :], None) in (-1, -3)
    good = [4096, 4096, 4096, 4096, 8, 2, 8, 0]
    for at, v in ((0, 0), (1, 0), (2, 0), (4, 7), (5, -1), (5, BIG), (6, -2), (7, 7)):
        assert lib.advopt_preference_loss_grad(*good[:at], v, *good[at + 1 :], None) in (-1, -3)


def test_work_sizes():
    from advanced_optimizers_b200 import _lib as L
    lib = L.lib()
    assert lib.advopt_embedding_grad_work(0, 8, 0) == 0 and lib.advopt_embedding_grad_work(256, 8, 0) == 0
    assert lib.advopt_embedding_grad_work(257, 8, 1) == 4 * 1040 + 33 * 2 * 8 * 4
    assert lib.advopt_embedding_grad_work(1 << 17, 8, 0) == 4 * (4 << 17) + (1 << 12) * 2 * 8 * 4
    assert lib.advopt_token_logprobs_work(500, 3000, 1) == 0 and lib.advopt_token_logprobs_work(500, 3200, 1) == 500 * 2 * 8
    assert lib.advopt_token_logprobs_work(148, 8193, 0) == 0 and lib.advopt_token_logprobs_work(149, 8193, 0) == 149 * 6 * 8
    assert lib.advopt_policy_loss_work(3, 1025) == 3 * 9 * 16 and lib.advopt_policy_loss_work(3, 0) == 0
    assert lib.advopt_policy_loss_work(3000, 1025) == 3000 * 2 * 16
    assert lib.advopt_preference_loss_work(3, 1024) == 6 * 8 * 8 + 6 * 16 and lib.advopt_preference_loss_work(3, 0) == 6 * 16
    assert lib.advopt_layer_norm_grad_work(0, 8) == 0 and lib.advopt_layer_norm_grad_work(5, 4096) == 5 * 2 * 4096 * 4




def _on_gpu(monkeypatch):
    """CPU tensors pass the device checks, so that the checks behind them can be tested here."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))


def test_refusals_behind_the_device_check(monkeypatch):
    import advanced_optimizers_b200 as A
    _on_gpu(monkeypatch)
    x, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    h, flags = torch.zeros(4, 8, dtype=torch.float16), torch.zeros(4, 8, dtype=torch.bool)
    cases = [
        (NotImplementedError, "not supported", lambda: A.embedding(ids, h)),
        (ValueError, "finite", lambda: A.embedding(ids, x, scale=NAN)),
        (ValueError, "padding_idx", lambda: A.embedding(ids, x, padding_idx=4)),
        (ValueError, "padding_idx", lambda: A.embedding(ids, x, padding_idx=-5)),
        (NotImplementedError, "not supported", lambda: A.layer_norm(h)),
        (NotImplementedError, "not supported", lambda: A.layer_norm(x, h[0])),
        (ValueError, "weight and bias are", lambda: A.layer_norm(x, x[0, :7])),
        (ValueError, "share a dtype", lambda: A.layer_norm(x, x[0], x[0].bfloat16())),
        (ValueError, "eps", lambda: A.layer_norm(x, eps=-1e-5)),
        (ValueError, "eps", lambda: A.layer_norm(x, eps=NAN)),
        (ValueError, "rows of 1", lambda: A.layer_norm(x[:, :0])),
        (NotImplementedError, "not supported", lambda: A.token_logprobs(h, ids)),
        (ValueError, "temperature", lambda: A.token_logprobs(x, ids, temperature=0)),
        (ValueError, "temperature", lambda: A.token_logprobs(x, ids, temperature=NAN)),
        (ValueError, "rows of 1", lambda: A.token_logprobs(x[:, :0], ids)),
        (ValueError, "64 bits", lambda: A.token_logprobs(x, ids, ignore_index=1 << 63)),
        (NotImplementedError, "not supported", lambda: A.policy_loss(h, h, h)),
        (ValueError, "dtype", lambda: A.policy_loss(x, h, x)),
        (ValueError, "shape", lambda: A.policy_loss(x, x[:, :7], x)),
        (ValueError, "advantages are", lambda: A.policy_loss(x, x, x[0])),
        (ValueError, "advantages are", lambda: A.policy_loss(x, x, x[:, :1])),
        (ValueError, "mask", lambda: A.policy_loss(x, x, x, x)),
        (ValueError, "mask", lambda: A.policy_loss(x, x, x, flags[:3])),
        (ValueError, "clip", lambda: A.policy_loss(x, x, x, clip=(1.1, 0.2))),
        (ValueError, "clip", lambda: A.policy_loss(x, x, x, clip=(0.2, -0.1))),
        (ValueError, "clip", lambda: A.policy_loss(x, x, x, clip=(0.2,))),
        (ValueError, "kl_weight", lambda: A.policy_loss(x, x, x, ref_logprobs=x, kl_weight=NAN)),
        (ValueError, "ref_logprobs", lambda: A.policy_loss(x, x, x, kl_weight=0.1)),
        (ValueError, "average", lambda: A.policy_loss(x, x, x, average="rows")),
        (ValueError, "even number", lambda: A.preference_loss(x[:3])),
        (ValueError, "even number", lambda: A.preference_loss(x[:0])),
        (ValueError, "beta", lambda: A.preference_loss(x, beta=NAN)),
        (ValueError, "label_smoothing", lambda: A.preference_loss(x, label_smoothing=1.5)),
        (ValueError, "shape", lambda: A.preference_loss(x, x[:2])),
        (ValueError, "mask", lambda: A.preference_loss(x, x, flags[:2])),
    ]
    for kind, match, call in cases:
        with pytest.raises(kind, match=match):
            call()


def test_a_saved_tensor_that_a_hook_changed_is_refused():
    from advanced_optimizers_b200._device import saved
    t = torch.zeros(3, 4)
    assert saved(t, "input", torch.float32, (3, 4), t.device) is t
    assert saved(t.t(), "input", torch.float32, (4, 3), t.device).is_contiguous()
    for dtype, shape, device in ((torch.int64, (3, 4), t.device), (torch.float32, (4, 3), t.device), (torch.float32, (3, 4), torch.device("meta"))):
        with pytest.raises(RuntimeError, match="hook on saved tensors"):
            saved(t, "input", dtype, shape, device)


def test_rows_that_are_read_as_they_lie():
    from advanced_optimizers_b200._device import rows_of
    from advanced_optimizers_b200.losses import _strided
    x = torch.arange(120.0).view(10, 12)
    for t, pitch in ((x, 12), (x[:, 3:7], 12), (x[::2], 24), (x[:1, 2:9], 7), (x[:, :1], 12)):
        got, ld = rows_of(t)
        assert got.data_ptr() == t.data_ptr() and ld == pitch
    for t in (x.t(), x[:1].expand(5, 12), x[:, ::2], x[0].as_strided((4, 6), (3, 1))):
        got, ld = rows_of(t)
        assert got.is_contiguous() and torch.equal(got, t) and ld == t.shape[1]
    y = torch.arange(240.0).view(2, 10, 12)
    for t in (y, y[:, :-1], y[:, 1:, 2:9], y[:1].expand(3, 10, 12), y[0], y.transpose(0, 1)):
        got, inner, outer, pitch = _strided(t)
        assert got.data_ptr() == t.data_ptr()
        for r in range(t[..., 0].numel()):
            at = r // inner * outer + r % inner * pitch
            assert torch.equal(got.as_strided((t.shape[-1],), (1,), got.storage_offset() + at), t.reshape(-1, t.shape[-1])[r])


def test_every_gpu_that_may_report_an_error_is_waited_for(monkeypatch):
    """Two GPUs' calls share a word: a check with either of them current waits for both."""
    import numpy as np
    from advanced_optimizers_b200 import _device, embeddings, fp8

    class Word:
        array = np.zeros(1, dtype=np.int32)
        numpy = lambda self: self.array  # noqa: E731
        data_ptr = lambda self: self.array.ctypes.data  # noqa: E731

    waited = []

    def synchronize(device=None):
        waited.append(device)
        if device == torch.device("cuda", 1):
            Word.array[0] = 1   # its kernel reports while it is waited for

    monkeypatch.setattr(torch, "zeros", lambda *a, **k: Word())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "synchronize", synchronize)
    for module, name, check in ((embeddings, "INDEX_ERRORS", embeddings.check_index_errors), (fp8, "_ERR", fp8.check_fp8_errors)):
        word = _device.ErrorWord()
        monkeypatch.setattr(module, name, word)
        check()   # nothing to wait for
        for index in (0, 1, 0):
            assert word.pointer(torch.device("cuda", index)) == Word.array.ctypes.data
        del waited[:]
        with pytest.raises(_device.L.AdvOptError):
            check()
        assert set(waited) == {torch.device("cuda", 0), torch.device("cuda", 1)} and Word.array[0] == 0


def test_numbers_that_float32_does_not_hold_are_refused(monkeypatch):
    import advanced_optimizers_b200 as A
    _on_gpu(monkeypatch)
    x, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for scale in (1e39, -1e39, 3.4028236e38):
        with pytest.raises(ValueError, match="scale"):
            A.embedding(ids, x, scale=scale)
    for eps in (1e39, 1e-50):   # the second would act as 0
        with pytest.raises(ValueError, match="eps"):
            A.layer_norm(x, eps=eps)


def test_layer_norm_s_sums_have_room_for_every_way_to_take_a_row():
    """A row of partial sums for each CTA: eight rows a CTA where warps take them, whatever their type and alignment, else one, until there
    is a CTA for each SM; then four times as many rows; never more than 1184."""
    from advanced_optimizers_b200 import _lib as L
    parts = lambda rows, cols: L.lib().advopt_layer_norm_grad_work(rows, cols) / (2 * cols * 4)  # noqa: E731
    for cols in (769, 776, 1000, 1023, 1024, 1032, 2048):
        assert [parts(r, cols) for r in (1, 7, 100, 148, 500, 1000, 4096, 100000)] == [1, 7, 100, 148, 148, 250, 1024, 1184]
    for cols in (1, 500, 700):
        assert [parts(r, cols) for r in (1, 7, 100, 1000, 4096, 100000)] == [1, 7, 13, 125, 148, 1184]
    for cols in (8193, 16384, 65536):
        assert [parts(r, cols) for r in (1, 98, 5000)] == [1, 98, 98]
    assert [parts(r, 70001) for r in (1, 100, 5000)] == [1, 13, 32]
