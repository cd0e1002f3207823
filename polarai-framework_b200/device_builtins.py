"""The builtins on torch CUDA tensors, under the reference's native kernel names.

`DeviceBuiltins` launches on torch's current stream with device tensors (what
the benchmark times); `HostBuiltins` has the oracle's call signatures - numpy in,
numpy out - and moves the data through the device, for the parity tests.
torch is used for device memory and streams only.

Each builtin first goes to the native binding (capi.binding), which checks its tensors
and launches without the interpreter; what that declines - tensors it would reject, a failing
call - runs the checked path below it, which raises.  An input may be longer than the result and a result
tensor larger than what is written; what would be read or written outside a tensor is a ValueError.
"""
import ctypes
import numbers

import numpy as np
import torch

from .capi import AdamwOptions, AdamwTensor, MuonOptions, MuonTensor, PolicyBatch, PolicyOptions, PreferenceOptions, binding, lib


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _stream(t):
    """torch's current stream ON THE TENSOR'S DEVICE (not on whatever device is current)."""
    return torch.cuda.current_stream(t.device).cuda_stream


def _chk(*ts):
    for t in ts:
        if not (t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()):
            raise ValueError("builtins take contiguous float32 CUDA tensors")


def _long_enough(n, *ts):
    for t in ts:
        if t.numel() < n:
            raise ValueError(f"a tensor of {t.numel()} elements where the builtin takes {n}")


def _chk_rows(*ts):
    """The tensors of a builtin on rows that are not None: as _chk, and all on one device."""
    _chk(*ts)
    _same_device(*ts)


def _same_device(*ts):
    if any(t.device != ts[0].device for t in ts):
        raise ValueError("the tensors of one call lie on one device")


def _exactly(what, n, *ts):
    for t in ts:
        if t is not None and t.numel() != n:
            raise ValueError(f"{what}: a tensor of {t.numel()} elements where {n} are taken")


_ID_TYPES = {torch.float32: 0, torch.int32: 1, torch.int64: 2}


def _matrix(t):
    """Its rows, their length and how far they lie apart."""
    if not (t.is_cuda and t.dtype == torch.float32 and t.dim() == 2 and (t.shape[1] <= 1 or t.stride(1) == 1)
            and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1])):
        raise ValueError("logits are float32 CUDA matrices of contiguous rows")
    rows, cols = t.shape
    return rows, cols, (cols if rows <= 1 else t.stride(0))


def _ids(t):
    if not (t.is_cuda and t.is_contiguous() and t.dtype in _ID_TYPES):
        raise ValueError("ids are contiguous CUDA tensors of float32, int32 or int64")
    return _ID_TYPES[t.dtype]


def _present(*ts):
    return [t for t in ts if t is not None]


def _packed(what, ids, offsets, *ts):
    """The tokens and the sequences of a batch, and how its ids and offsets are held."""
    _chk(*ts)
    if _ids(ids) != _ids(offsets):
        raise ValueError(f"{what}: ids and offsets are of one type")
    _same_device(ids, offsets, *ts)
    if offsets.numel() < 1:
        raise ValueError(f"{what}: offsets are one more than the sequences")
    return ids.numel(), offsets.numel() - 1, _ids(ids)


class DeviceBuiltins:
    def __init__(self):
        if not torch.cuda.is_available():
            raise RuntimeError("no CUDA device: the PolarAI B200 builtins have no CPU path")
        self.lib = lib()
        self._native = binding()

    def ffill(self, pattern, out):
        if not self._native.ffill(pattern, out):
            _chk(out)
            self.lib.call("polar_b200_ffill", float(pattern), _ptr(out), out.numel(), _stream(out))
        return out

    def fcopy(self, a, out):
        if not self._native.fcopy(a, out):
            _chk(a, out)
            _long_enough(out.numel(), a)
            self.lib.call("polar_b200_fcopy", _ptr(a), _ptr(out), out.numel(), _stream(out))
        return out

    def fadd(self, a, sa, b, sb, out):
        if not self._native.fadd(a, sa, b, sb, out):
            _chk(a, b, out)
            _long_enough(out.numel(), a, b)
            self.lib.call("polar_b200_fadd", _ptr(a), float(sa), _ptr(b), float(sb), _ptr(out), out.numel(),
                          _stream(out))
        return out

    def fmul(self, a, b, out):
        if not self._native.fmul(a, b, out):
            _chk(a, b, out)
            _long_enough(out.numel(), a, b)
            self.lib.call("polar_b200_fmul", _ptr(a), _ptr(b), _ptr(out), out.numel(), _stream(out))
        return out

    def fdivide(self, a, b, out):
        if not self._native.fdivide(a, b, out):
            _chk(a, b, out)
            _long_enough(out.numel(), a, b)
            self.lib.call("polar_b200_fdivide", _ptr(a), _ptr(b), _ptr(out), out.numel(), _stream(out))
        return out

    def fsigmoid(self, a, out, clamp=True):
        if not (self._native.fsigmoid if clamp else self._native.fsigmoid_unclamped)(a, out):
            _chk(a, out)
            _long_enough(out.numel(), a)
            name = "polar_b200_fsigmoid" if clamp else "polar_b200_fsigmoid_unclamped"
            self.lib.call(name, _ptr(a), _ptr(out), out.numel(), _stream(out))
        return out

    def flogloss(self, predicted, ground_truth, out):
        if not self._native.flogloss(predicted, ground_truth, out):
            _chk(predicted, ground_truth, out)
            _long_enough(out.numel(), predicted, ground_truth)
            self.lib.call("polar_b200_flogloss", _ptr(predicted), _ptr(ground_truth), _ptr(out), out.numel(),
                          _stream(out))
        return out

    def fmulconcat(self, gradient, local, out):
        if not self._native.fmulconcat(gradient, local, out):
            _chk(gradient, local, out)
            _long_enough(out.numel(), local)
            self.lib.call("polar_b200_fmulconcat", _ptr(gradient), _ptr(local), _ptr(out), out.numel(), _stream(out))
        return out

    def frelu(self, a, out):
        if not self._native.frelu(a, out):
            _chk(a, out)
            _long_enough(out.numel(), a)
            self.lib.call("polar_b200_frelu", _ptr(a), _ptr(out), out.numel(), _stream(out))
        return out

    def fsoftmax(self, a, out):
        if not self._native.fsoftmax(a, out):
            _chk(a, out)
            _long_enough(out.numel(), a)
            self.lib.call("polar_b200_fsoftmax", _ptr(a), _ptr(out), out.numel(), None, 0, _stream(out))
        return out

    def fpool(self, a, window, stride, out):
        if not self._native.fpool(a, window[0], window[1], stride[0], stride[1], out):
            _chk(a, out)
            h, w = a.shape
            if 0 < window[0] <= h and 0 < window[1] <= w and stride[0] > 0 and stride[1] > 0:   # (else the library's error)
                _long_enough(((h - window[0]) // stride[0] + 1) * ((w - window[1]) // stride[1] + 1), out)
            self.lib.call("polar_b200_fpool", _ptr(a), h, w, window[0], window[1], stride[0], stride[1], _ptr(out),
                          _stream(out))
        return out

    def fconv2d(self, a, kernel, out):
        if not self._native.fconv2d(a, kernel, out):
            _chk(a, kernel, out)
            h, w = a.shape
            kh, kw = kernel.shape
            _long_enough(max(h - kh + 1, 0) * max(w - kw + 1, 0), out)
            self.lib.call("polar_b200_fconv2d", _ptr(a), h, w, _ptr(kernel), kh, kw, _ptr(out), _stream(out))
        return out

    def ftranspose(self, a, out):
        if not self._native.ftranspose(a, out):
            _chk(a, out)
            rows, cols = a.shape
            _long_enough(rows * cols, out)
            self.lib.call("polar_b200_ftranspose", _ptr(a), rows, cols, _ptr(out), _stream(out))
        return out

    def fslice(self, a, index, out):
        _chk(a, out)
        if 0 <= int(index) < a.shape[0]:                     # (else the library's error)
            _long_enough((int(index) + 1) * out.numel(), a)
        self.lib.call("polar_b200_fslice", _ptr(a), a.shape[0], out.numel(), int(index), _ptr(out), _stream(out))
        return out

    def fsum(self, a, acc):
        """Adds sum(a) to the float64 one-element tensor `acc`."""
        _chk(a)
        self.lib.call("polar_b200_fsum", _ptr(a), _ptr(acc), a.numel(), _stream(a))
        return acc

    def fmatmul(self, tl, tr, left, right, out):
        if not self._native.fmatmul(tl, tr, left, right, out):
            _chk(left, right, out)
            m, n, k = matmul_dims(tl, tr, left.shape, right.shape)
            if tuple(out.shape) != (m, n):
                raise ValueError(f"out must be [{m},{n}]")
            self.lib.call("polar_b200_fmatmul", int(tl), int(tr), m, n, k, _ptr(left), _ptr(right), _ptr(out),
                          None, 0, _stream(out))
        return out

    def fmatmul_ffma(self, tl, tr, left, right, out):
        _chk(left, right, out)
        m, n, k = matmul_dims(tl, tr, left.shape, right.shape)
        _long_enough(m * n, out)
        self.lib.call("polar_b200_fmatmul_ffma", int(tl), int(tr), m, n, k, _ptr(left), _ptr(right),
                      _ptr(out), _stream(out))
        return out

    def fmatmul_tc(self, tl, tr, left, right, out, tile_n=256, slab_k=16, passes=3, write_hi=0, splits=1):
        _chk(left, right, out)
        m, n, k = matmul_dims(tl, tr, left.shape, right.shape)
        _long_enough(m * n, out)
        self.lib.call("polar_b200_fmatmul_tc", int(tl), int(tr), m, n, k, _ptr(left), _ptr(right),
                      _ptr(out), tile_n, slab_k, passes, write_hi, splits, _stream(out))
        return out

    def flayernorm(self, x, gamma, beta, eps, out, mean=None, rstd=None):
        """out = (x - mean) * rstd * gamma + beta over the last dimension of x; gamma, beta, mean, rstd may be None."""
        if not self._native.flayernorm(x, gamma, beta, eps, out, mean, rstd):
            _chk_rows(*_present(x, gamma, beta, out, mean, rstd))
            cols = x.shape[-1] if x.dim() else 0
            rows = x.numel() // cols if cols else 0
            _exactly("flayernorm", x.numel(), out)
            _exactly("flayernorm", cols, gamma, beta)
            _exactly("flayernorm", rows, mean, rstd)
            self.lib.call("polar_b200_flayernorm", _ptr(x), _ptr(gamma), _ptr(beta), float(eps), rows, cols, _ptr(out), _ptr(mean),
                          _ptr(rstd), _stream(out))
        return out

    def flayernorm_grad(self, gradient, x, gamma, mean, rstd, dx, dgamma=None, dbeta=None):
        """The gradients at flayernorm's x, gamma and beta (the last two may be None, as gamma may); mean, rstd are flayernorm's."""
        if not self._native.flayernorm_grad(gradient, x, gamma, mean, rstd, dx, dgamma, dbeta):
            _chk_rows(*_present(gradient, x, gamma, mean, rstd, dx, dgamma, dbeta))
            cols = x.shape[-1] if x.dim() else 0
            rows = x.numel() // cols if cols else 0
            _exactly("flayernorm_grad", x.numel(), gradient, dx)
            _exactly("flayernorm_grad", cols, gamma, dgamma, dbeta)
            _exactly("flayernorm_grad", rows, mean, rstd)
            self.lib.call("polar_b200_flayernorm_grad", _ptr(gradient), _ptr(x), _ptr(gamma), _ptr(mean), _ptr(rstd), rows, cols,
                          _ptr(dx), _ptr(dgamma), _ptr(dbeta), None, 0, _stream(dx))
        return dx

    def flogprob(self, logits, ids, logprob, entropy=None, logsumexp=None, top_ids=None, top_logprob=None):
        """Per row of logits: the log probability of its id (0 where the id is below zero), the entropy, log(sum(exp)), and the
        likeliest alternatives [rows, top] (up to 32; ids of the type of `ids`).  What is None is left out."""
        if not self._native.flogprob(logits, ids, logprob, entropy, logsumexp, top_ids, top_logprob):
            rows, classes, pitch = _matrix(logits)
            some = _present(logprob, entropy, logsumexp, top_logprob)
            if some:
                _chk(*some)
            kinds = {_ids(t) for t in _present(ids, top_ids)}
            _same_device(logits, *some, *_present(ids, top_ids))
            if len(kinds) > 1:
                raise ValueError("flogprob: top_ids are of the type of ids")
            _exactly("flogprob", rows, ids, logprob, entropy, logsumexp)
            tops = {tuple(t.shape) for t in _present(top_ids, top_logprob)}
            if len(tops) > 1 or any(len(s) != 2 or s[0] != rows for s in tops):
                raise ValueError("flogprob: alternatives are [rows, top]")
            if logprob is not None and ids is None:
                raise ValueError("flogprob: a log probability needs ids")
            self.lib.call("polar_b200_flogprob", _ptr(logits), rows, classes, pitch, _ptr(ids), kinds.pop() if kinds else 2,
                          _ptr(logprob), _ptr(entropy), _ptr(logsumexp), tops.pop()[1] if tops else 0, _ptr(top_ids), _ptr(top_logprob),
                          _stream(logits))
        return logprob

    def flogprob_grad(self, logits, ids, logsumexp, entropy, g_logprob, g_entropy, dlogits):
        """The gradient at the logits of sum(g_logprob * logprob + g_entropy * entropy); entropy and g_entropy may be None."""
        if not self._native.flogprob_grad(logits, ids, logsumexp, entropy, g_logprob, g_entropy, dlogits):
            rows, classes, pitch = _matrix(logits)
            drows, dclasses, dpitch = _matrix(dlogits)
            given = _present(logsumexp, entropy, g_logprob, g_entropy)
            _chk(*given)
            kind = _ids(ids)
            _same_device(logits, dlogits, ids, *given)
            if (drows, dclasses) != (rows, classes):
                raise ValueError("flogprob_grad: dlogits has the shape of logits")
            _exactly("flogprob_grad", rows, ids, *given)
            if g_entropy is not None and entropy is None:
                raise ValueError("flogprob_grad: the entropy's gradient needs the entropy")
            self.lib.call("polar_b200_flogprob_grad", _ptr(logits), rows, classes, pitch, _ptr(ids), kind, _ptr(logsumexp), _ptr(entropy),
                          _ptr(g_logprob), _ptr(g_entropy), _ptr(dlogits), dpitch, _stream(dlogits))
        return dlogits

    def fadamw(self, weights, gradients, first, second, first_scales=None, second_scales=None, *, step=0, lr=0.0, beta1=0.9,
               beta2=0.999, eps=1e-8, weight_decay=0.01, schedule=None):
        """One AdamW step over lists of tensors, in place.  `first` and `second` are the moments: float32 of the weights' sizes or,
        with scales, float8_e4m3fn (or uint8) codes of the weights' sizes, whose scales are float32 of ceil(n / 128).
        weight_decay: one for all, or a list.  The number of the step (from 1) and lr come from the call or, for steps that are
        captured, from `schedule`, a device tensor of the two."""
        decays = [weight_decay] * len(weights) if isinstance(weight_decay, numbers.Real) else weight_decay
        if not self._native.fadamw(weights, gradients, first, second, first_scales, second_scales, step, lr, beta1, beta2, eps, decays,
                                   schedule):
            lists = _present(weights, gradients, first, second, first_scales, second_scales)
            if (first_scales is None) != (second_scales is None) or any(len(x) != len(weights) for x in [*lists, decays]):
                raise ValueError("fadamw: lists of one length, and scales for both moments or neither")
            eight = first_scales is not None
            tensors = (AdamwTensor * len(weights))()
            for t, decay, w, g, m, v, *scales in zip(tensors, decays, *lists):
                _chk(w, g, *scales, *(() if eight else (m, v)))
                if eight and not all(x.is_cuda and x.is_contiguous() and x.dtype in (torch.float8_e4m3fn, torch.uint8) for x in (m, v)):
                    raise ValueError("fadamw: moments in 8 bits are contiguous float8_e4m3fn or uint8 CUDA tensors")
                _same_device(weights[0], w, g, m, v, *scales)
                _exactly("fadamw", w.numel(), g, m, v)
                _exactly("fadamw", -(-w.numel() // 128), *scales)
                t.weights, t.gradient, t.first, t.second = (x.data_ptr() for x in (w, g, m, v))
                if eight:
                    t.first_scales, t.second_scales = (x.data_ptr() for x in scales)
                t.count, t.weight_decay = w.numel(), float(decay)
            if schedule is not None:
                _chk(schedule)
                _exactly("fadamw", 2, schedule)
                _same_device(schedule, *weights[:1])
            if int(step) < 0:
                raise ValueError("fadamw: steps count from 1")
            if weights:
                options = AdamwOptions(float(lr), float(beta1), float(beta2), float(eps), int(step), _ptr(schedule))
                self.lib.call("polar_b200_fadamw", tensors, len(weights), ctypes.byref(options), _stream(weights[0]))
        return weights

    def fmuon(self, weights, gradients, momenta, *, lr=0.0, momentum=0.95, nesterov=True, steps=5, weight_decay=0.0, scale=None,
              coefficients=(3.4445, -4.7750, 2.0315), schedule=None):
        """One step of orthogonalised momentum over lists of matrices - tensors [rows, cols], or [..., rows, cols] of several, each by
        itself - in place; gradients and momenta have their shape.  weight_decay and scale, by which the update is multiplied: one for all, or a list; no scale: sqrt(rows / cols) where
        that is above 1.  lr comes from the call or, for steps that are captured, from `schedule`, fadamw's device tensor of the step's number and lr."""
        if not self._native.fmuon(weights, gradients, momenta, lr, momentum, bool(nesterov), steps, weight_decay, scale, *coefficients, schedule):
            decays = [weight_decay] * len(weights) if isinstance(weight_decay, numbers.Real) else weight_decay
            scales = ([scale] * len(weights) if isinstance(scale, numbers.Real) else scale if scale is not None else
                      [max(1.0, w.shape[-2] / max(w.shape[-1], 1)) ** 0.5 if len(w.shape) >= 2 else 1.0 for w in weights])
            if any(len(x) != len(weights) for x in (gradients, momenta, decays, scales)):
                raise ValueError("fmuon: lists of one length")
            tensors = (MuonTensor * len(weights))()
            for t, w, g, m, decay, s in zip(tensors, weights, gradients, momenta, decays, scales):
                _chk(w, g, m)
                _same_device(weights[0], w, g, m)
                _exactly("fmuon", w.numel(), g, m)
                if len(w.shape) < 2:
                    raise ValueError("fmuon: weights are matrices (vectors are for fadamw)")
                if any(tuple(x.shape[-2:]) != tuple(w.shape[-2:]) for x in (g, m)):
                    raise ValueError("fmuon: a gradient and a momentum have the shape of their weights")
                t.weights, t.gradient, t.momentum = (x.data_ptr() for x in (w, g, m))
                t.rows, t.cols = w.shape[-2:]
                t.matrices = w.numel() // (t.rows * t.cols) if t.rows and t.cols else 0
                t.weight_decay, t.scale = float(decay), float(s)
            if schedule is not None:
                _chk(schedule)
                _exactly("fmuon", 2, schedule)
                _same_device(schedule, *weights[:1])
            if weights:
                options = MuonOptions(float(lr), float(momentum), int(bool(nesterov)), max(int(steps), 0), *(float(c) for c in coefficients), _ptr(schedule))
                need = self.lib.cdll.polar_b200_fmuon_workspace_bytes(tensors, len(weights))
                workspace = torch.empty(need, dtype=torch.uint8, device=weights[0].device) if need else None
                self.lib.call("polar_b200_fmuon", tensors, len(weights), ctypes.byref(options), _ptr(workspace), need, _stream(weights[0]))
        return weights

    def fpolicy_loss(self, logprob, old_logprob, advantage, ids, offsets, loss, g_logprob=None, g_entropy=None, *, reference=None, entropy=None,
                     clip_low=0.2, clip_high=0.2, kl_weight=0.0, entropy_weight=0.0, by_sequence=False, advantage_per_token=False, count=0.0):
        """The clipped policy loss of packed sequences into loss[5] - the loss and, as means over the tokens that count, surrogate, KL term,
        entropy, share of clipped tokens - and its gradients at the log probabilities and the entropies.  Sequence s has the tokens
        [offsets[s], offsets[s + 1]), a token with an id below zero does not count; `reference`: log probabilities for the KL term.
        The mean goes over the tokens or, by_sequence, over the sequences' means; `count` above zero is divided by in place of their number.
        The advantage is one for each sequence or, advantage_per_token, for each token.  Gradients before the first sequence and behind the last one
        are left as they are."""
        if not self._native.fpolicy_loss(logprob, old_logprob, reference, entropy, advantage, ids, offsets, advantage_per_token, clip_low, clip_high,
                                         kl_weight, entropy_weight, count, by_sequence, loss, g_logprob, g_entropy):
            arrays = _present(logprob, old_logprob, reference, entropy, g_logprob, g_entropy)
            tokens, sequences, kind = _packed("fpolicy_loss", ids, offsets, loss, advantage, *arrays)
            _exactly("fpolicy_loss", tokens, *arrays)
            _exactly("fpolicy_loss", tokens if advantage_per_token else sequences, advantage)
            _exactly("fpolicy_loss", 5, loss)
            if g_entropy is not None and entropy is None:
                raise ValueError("fpolicy_loss: the entropy's gradient needs the entropy")
            batch = PolicyBatch(_ptr(logprob), _ptr(old_logprob), _ptr(reference), _ptr(entropy), _ptr(advantage), _ptr(ids), _ptr(offsets), kind,
                                int(bool(advantage_per_token)), tokens, sequences)
            options = PolicyOptions(float(clip_low), float(clip_high), float(kl_weight), float(entropy_weight), float(count), int(bool(by_sequence)))
            self.lib.call("polar_b200_fpolicy_loss", ctypes.byref(batch), ctypes.byref(options), _ptr(loss), _ptr(g_logprob), _ptr(g_entropy),
                          None, 0, _stream(loss))
        return loss

    def fpreference_loss(self, logprob, ids, offsets, loss, rewards=None, g_logprob=None, *, reference=None, beta=0.1, smoothing=0.0, margin=0.0,
                         average=False, count=0.0):
        """The loss of pairs of packed sequences, 2i the chosen and 2i + 1 the rejected one, into loss[3] - the loss, the share of pairs in the
        right order, their mean difference - with the sequences' rewards, beta times the sum (average: the mean) of logprob - reference over
        the tokens that count, and the loss's gradient at the log probabilities, which stays as it is before the first sequence and behind the last one.
        `count` above zero is divided by in place of the pairs' number."""
        if not self._native.fpreference_loss(logprob, reference, ids, offsets, beta, smoothing, margin, count, average, loss, rewards, g_logprob):
            arrays = _present(logprob, reference, g_logprob)
            tokens, sequences, kind = _packed("fpreference_loss", ids, offsets, loss, *_present(rewards), *arrays)
            if sequences % 2:
                raise ValueError("fpreference_loss: pairs of sequences")
            _exactly("fpreference_loss", tokens, *arrays)
            _exactly("fpreference_loss", sequences, rewards)
            _exactly("fpreference_loss", 3, loss)
            options = PreferenceOptions(float(beta), float(smoothing), float(margin), float(count), int(bool(average)))
            self.lib.call("polar_b200_fpreference_loss", _ptr(logprob), _ptr(reference), _ptr(ids), _ptr(offsets), kind, tokens, sequences // 2,
                          ctypes.byref(options), _ptr(loss), _ptr(rewards), _ptr(g_logprob), None, 0, _stream(loss))
        return loss

    def device_status(self):
        return int(self.lib.cdll.polar_b200_device_status())


def matmul_dims(tl, tr, lshape, rshape):
    m = lshape[1] if tl else lshape[0]
    k = lshape[0] if tl else lshape[1]
    n = rshape[0] if tr else rshape[1]
    k2 = rshape[1] if tr else rshape[0]
    if k != k2:
        raise ValueError(f"inner dimensions differ: {k} vs {k2}")
    return int(m), int(n), int(k)


class HostBuiltins:
    """numpy in / numpy out, every call through the device."""

    def __init__(self, device="cuda:0"):
        self.dev = torch.device(device)
        self.d = DeviceBuiltins()

    def _up(self, a):
        return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(self.dev)

    def _down(self, t):
        torch.cuda.synchronize(self.dev)
        return t.cpu().numpy()

    def ffill(self, pattern, n):
        return self._down(self.d.ffill(pattern, torch.empty(n, device=self.dev)))

    def fcopy(self, a):
        a = self._up(a)
        return self._down(self.d.fcopy(a, torch.empty_like(a)))

    def fadd(self, a, sa, b, sb):
        a, b = self._up(a), self._up(b)
        return self._down(self.d.fadd(a, sa, b, sb, torch.empty_like(a)))

    def fmul(self, a, b):
        a, b = self._up(a), self._up(b)
        return self._down(self.d.fmul(a, b, torch.empty_like(a)))

    def fdivide(self, a, b):
        a, b = self._up(a), self._up(b)
        return self._down(self.d.fdivide(a, b, torch.empty_like(a)))

    def fsigmoid(self, a, clamp=True):
        a = self._up(a)
        return self._down(self.d.fsigmoid(a, torch.empty_like(a), clamp))

    def flogloss(self, p, y):
        p, y = self._up(p), self._up(y)
        return self._down(self.d.flogloss(p, y, torch.empty_like(p)))

    def fmulconcat(self, g, l):
        g, l = self._up(g), self._up(l)
        return self._down(self.d.fmulconcat(g, l, torch.empty_like(l)))

    def frelu(self, a):
        a = self._up(a)
        return self._down(self.d.frelu(a, torch.empty_like(a)))

    def fsoftmax(self, a):
        a = self._up(a)
        return self._down(self.d.fsoftmax(a, torch.empty_like(a)))

    def fpool(self, a, window, stride):
        a = self._up(a)
        h, w = a.shape
        out = torch.empty(((h - window[0]) // stride[0] + 1, (w - window[1]) // stride[1] + 1), device=self.dev)
        return self._down(self.d.fpool(a, window, stride, out))

    def fconv2d(self, a, kernel):
        a, kernel = self._up(a), self._up(kernel)
        out = torch.empty((a.shape[0] - kernel.shape[0] + 1, a.shape[1] - kernel.shape[1] + 1), device=self.dev)
        return self._down(self.d.fconv2d(a, kernel, out))

    def ftranspose(self, a):
        a = self._up(a)
        return self._down(self.d.ftranspose(a, torch.empty((a.shape[1], a.shape[0]), device=self.dev)))

    def fslice(self, a, index):
        a = self._up(a)
        return self._down(self.d.fslice(a, index, torch.empty(tuple(a.shape[1:]), device=self.dev)))

    def flayernorm(self, x, gamma, beta, eps):
        x, gamma, beta = self._up(x), self._up(gamma), self._up(beta)
        mean, rstd = (torch.empty(x.shape[:-1], device=self.dev) for _ in range(2))
        out = self.d.flayernorm(x, gamma, beta, eps, torch.empty_like(x), mean, rstd)
        return tuple(self._down(t) for t in (out, mean, rstd))

    def flayernorm_grad(self, gradient, x, gamma, mean, rstd):
        g, x, gamma, mean, rstd = (self._up(t) for t in (gradient, x, gamma, mean, rstd))
        dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(gamma)
        dx = self.d.flayernorm_grad(g, x, gamma, mean, rstd, torch.empty_like(x), dgamma, dbeta)
        return tuple(self._down(t) for t in (dx, dgamma, dbeta))

    def flogprob(self, logits, ids, top=0):
        x, ids = self._up(logits), torch.from_numpy(np.ascontiguousarray(ids, np.int64)).to(self.dev)
        lp, entropy, lse = (torch.empty(len(ids), device=self.dev) for _ in range(3))
        top_ids = torch.empty((len(ids), top), dtype=torch.int64, device=self.dev)
        top_lp = torch.empty((len(ids), top), device=self.dev)
        self.d.flogprob(x, ids, lp, entropy, lse, top_ids if top else None, top_lp if top else None)
        return tuple(self._down(t) for t in (lp, entropy, lse, top_ids, top_lp))

    def flogprob_grad(self, logits, ids, logsumexp, entropy, g_logprob, g_entropy):
        x, ids = self._up(logits), torch.from_numpy(np.ascontiguousarray(ids, np.int64)).to(self.dev)
        lse, h, g, gh = (None if t is None else self._up(t) for t in (logsumexp, entropy, g_logprob, g_entropy))
        return self._down(self.d.flogprob_grad(x, ids, lse, h, g, gh, torch.empty_like(x)))

    def fadamw(self, w, g, m, v, step, lr, beta1, beta2, eps, decay):
        w, g, m, v = (self._up(t).clone() for t in (w, g, m, v))
        self.d.fadamw([w], [g], [m], [v], step=step, lr=lr, beta1=beta1, beta2=beta2, eps=eps, weight_decay=decay)
        return tuple(self._down(t) for t in (w, m, v))

    def fmatmul(self, tl, tr, left, right, which="auto", **kw):
        l, r = self._up(left), self._up(right)
        m, n, k = matmul_dims(tl, tr, l.shape, r.shape)
        out = torch.empty((m, n), device=self.dev)
        fn = {"auto": self.d.fmatmul, "ffma": self.d.fmatmul_ffma, "tc": self.d.fmatmul_tc}[which]
        return self._down(fn(tl, tr, l, r, out, **kw))
