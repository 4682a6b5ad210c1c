"""Operators of the dense (bf16 / fp32) models as objects: packed matrices, norms, epilogues and prologues of their
launches (include/llamatov_b200_dense.h).

Matrices are packed with head sizes and row lengths padded to multiples of 8 with zeros, so kernels need no ragged edges.
"""
import ctypes

import torch

from . import _lib
from . import dev_residency as dr

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def pad8(n):
    return (n + 7) // 8 * 8


# --------------------------------------------------------------------------- packing helpers

def _head_rows(W, sizes, heads):
    """Rows of a projection laid out head by head, each head `sizes` = [(n, padded n), ...] consecutive pieces."""
    per = sum(n for n, _ in sizes)
    W = W.reshape(heads, per, *W.shape[1:])
    parts, r = [], 0
    for n, p in sizes:
        piece = W[:, r:r + n]
        r += n
        if p > n:
            piece = torch.cat([piece, piece.new_zeros((heads, p - n) + tuple(W.shape[2:]))], dim=1)
        parts.append(piece)
    out = torch.cat(parts, dim=1)
    return out.reshape(-1, *W.shape[2:])


def _head_cols(W, n, heads):
    """Columns of an output projection, each head's n padded to a multiple of 8."""
    return _head_rows(W.T.contiguous(), [(n, pad8(n))], heads).T.contiguous()


def _pad_cols(W, k):
    return W if W.shape[1] == k else torch.cat([W, W.new_zeros(W.shape[0], k - W.shape[1])], dim=1)


def _pad_rows(W, n):
    return W if W.shape[0] == n else torch.cat([W, W.new_zeros((n - W.shape[0],) + tuple(W.shape[1:]))], dim=0)


# --------------------------------------------------------------------------- launch helpers

class Linear:
    """A packed matrix on the device: rows() over token rows, row() for one token with the input made in the kernel."""

    def __init__(self, W, dtype):
        W = _pad_cols(W.to(dtype), pad8(W.shape[1])).contiguous()
        self.M, self.K = W.shape
        self.f32 = int(dtype == torch.float32)
        self.W = W.cuda()
        self.ptr = self.W.data_ptr()

    def rows(self, x, ldx, y, ldy, T, epi, M=None, first=0):
        """Outputs of the matrix rows from `first` on, M of them (gated: M gate rows, then M up rows)."""
        _lib.call("lt_dn_linear", self.ptr + first * self.K * self.W.element_size(), self.K, x, ldx, y, ldy, self.f32,
                  self.M - first if M is None else M, self.K, T, ctypes.byref(epi), 0, dr._stream())

    def row(self, pro, y, epi, M=None):
        _lib.call("lt_dn_gemv", self.ptr, self.K, y, self.f32, self.M if M is None else M, self.K, ctypes.byref(pro),
                  ctypes.byref(epi), dr._stream())


def epilogue(kind=_lib.DN_STORE, segs=(), bias=None, ls=None, out_f32=False, glu=None, tail_from=None):
    """segs: (end, activation name or None, scale) per output segment.  glu: (act, alpha, limit) of gated outputs.
    tail_from: outputs from there on go to an fp32 buffer (`with_tail`)."""
    e = _lib.DnEpilogue()
    e.kind, e.out_f32, e.nseg = kind, int(out_f32), len(segs)
    for i, (end, act, scale) in enumerate(segs):
        e.seg_end[i], e.seg_act[i], e.seg_scale[i] = end, _lib.DN_ACT[act], scale
    e.bias = None if bias is None else bias.data_ptr()
    e.ls = None if ls is None else ls.data_ptr()
    if glu is not None:
        e.glu_act, e.glu_alpha, e.glu_limit = glu
    if tail_from is not None:
        e.tail_from = tail_from
    return e


def with_tail(epi, tail, ld):
    """The epilogue with its fp32 tail at `tail`, row stride ld."""
    e = _lib.DnEpilogue.from_buffer_copy(epi)
    e.tail, e.ldtail = tail, ld
    return e


class Norm:
    """RMS norm over groups of `group` (padded) elements of which `count` are real; weight repeats every w_period.
    gate_first: a gate multiplies ahead of the norm.  seg = (n, padded n): groups of `count` real elements that do not
    follow the padded segments."""

    def __init__(self, w, count, group, eps, gate_first=False, seg=None):
        self.w = w.float().cuda().contiguous()
        self.count, self.group, self.eps = int(count), int(group), float(eps)
        self.gate_first = int(gate_first)
        self.seg, self.segp = seg or (0, 0)

    def prologue(self, x, gate=None):
        return _lib.DnPrologue(_lib.DN_IN_NORM, 0, self.group, self.count, self.eps, x, None, self.w.data_ptr(),
                               self.w.numel(), gate, self.gate_first, self.seg, self.segp)

    def rows(self, x, ldx, y, ldy, f32, T, N, gate=None, ldg=0, index=None):
        _lib.call("lt_dn_norm_rows", x, ldx, index, self.w.data_ptr(), self.w.numel(), gate, ldg, y, ldy, f32, T, N,
                  self.group, self.count, self.eps, self.gate_first, self.seg, self.segp, dr._stream())


def typed_input(x):
    return _lib.DnPrologue(_lib.DN_IN_TYPED, 0, 0, 0, 0.0, x, None, None, 0, None, 0, 0, 0)


def cast_input(x, n1, x2=None):
    return _lib.DnPrologue(_lib.DN_IN_CAST, n1, 0, 0, 0.0, x, x2, None, 0, None, 0, 0, 0)


# --------------------------------------------------------------------------- sparse feed-forwards

def _stream(home=None):
    """The current stream's handle, as dev_residency._stream, without the Stream object that it makes (3 us of a call's 8).  home:
    the device that the caller's own memory is on; a launch on another one is refused."""
    device = torch.cuda.current_device()
    if home is not None and home != device:
        raise ValueError(f"made on cuda:{home}, the current device is cuda:{device}")
    return torch._C._cuda_getCurrentRawStream(device)


def _here(t, what):
    """Launches go to the current device: an operand of another one is refused."""
    if t.device.type != "cuda" or t.device.index != torch.cuda.current_device():
        raise ValueError(f"{what} is on {t.device}, the current device is cuda:{torch.cuda.current_device()}")
    return t


def group_from(n):
    """Places from which on the products of n experts go expert by expert, and not place by place.  An expert's matrix is read once
    then, which pays when experts are hit more than once, but the order of the places and the rows in that order cost launches.  (bf16,
    us place by place / by expert, gate|up and then down: 64 experts of 1024 x 2048, 32 places 43 / 50 and 25 / 36, 48 57 / 53 and
    36 / 38, 64 75 / 59 and 39 / 41; 8 of 2048 x 2048, 8 places 26 / 32 and 15 / 26, 12 34 / 32 and 19 / 28, 16 40 / 33 and 21 / 28, 24
    52 / 33 and 30 / 29; 128 of 512 x 1024, 64 places 25 / 33 and 16 / 23.)"""
    return GROUP_FROM if GROUP_FROM is not None else max(14, 3 * n // 4)


GROUP_FROM = None       # a number: whatever the experts


class Router:
    """Choice of `top` of n experts for rows of fp32 scores, and the weights of the chosen (lt_dn_route)."""

    def __init__(self, n, top, score="softmax", bias=None, groups=1, top_groups=1, renorm=True, scale=1.0):
        if score not in _lib.DN_SCORE:
            raise ValueError(f"score {score!r}: known are {', '.join(sorted(_lib.DN_SCORE))}")
        if not (1 <= top <= 32 and 1 <= n <= 1024 and 1 <= groups <= 32 and n % groups == 0 and 1 <= top_groups <= groups
                and top <= n // groups * top_groups):
            raise ValueError(f"top {top} of {n} experts in {top_groups} of {groups} groups")
        if bias is not None and tuple(bias.shape) != (n,):
            raise ValueError(f"bias {tuple(bias.shape)} for {n} experts")
        self.n, self.top = n, top
        self.bias = None if bias is None else bias.float().cuda().contiguous()
        self.home = None if bias is None else self.bias.device.index
        self.desc = _lib.DnRouter(n, top, _lib.DN_SCORE[score], groups, top_groups, int(renorm), float(scale),
                                  None if bias is None else self.bias.data_ptr())
        self._ref = ctypes.byref(self.desc)

    def rows(self, logits, ld, ids, w, T):
        """ids int32 [T][top] and w fp32 [T][top] of T rows of logits."""
        _lib.call("lt_dn_route", logits, ld, ids, w, T, self._ref, _stream(self.home))


class Places:
    """Chosen experts of T tokens (ids int32 [T, top]) and, with `plan`, the order of the places by expert.  stream: the handle of
    the stream that `plan` was allocated on, None where its memory is the caller's to keep."""

    def __init__(self, ids, n, plan=None, stream=None):
        self.ids, self.n, self.buf, self.stream = ids, n, plan, stream
        self.T, self.top = ids.shape
        self.desc = _lib.DnChoice(ids.data_ptr(), None if plan is None else plan.data_ptr(), self.T, self.top, n)
        self.ref = ctypes.byref(self.desc)


class Experts:
    """A matrix per expert, [n, rows, columns], the columns a multiple of 8.  gated: rows are gate rows and as many up rows, and
    `hidden` stores their gated product; else `add_sum` adds the weighted sum of the chosen experts' outputs to fp32 rows.  glu: as
    in `epilogue`."""

    def __init__(self, W, gated, glu=(_lib.DN_GLU_GELU, 0.0, 0.0)):
        if W.dim() != 3 or W.dtype not in DTYPES.values():
            raise ValueError(f"matrices {tuple(W.shape)} of {W.dtype}")
        n, M, K = W.shape
        if gated and M % 2:
            raise ValueError(f"{M} gate and up rows")
        if K % 8:                # columns added here would be read of the caller's rows too, where nothing has written them
            raise ValueError(f"{K} columns: they must be a multiple of 8 (zeros in the matrices and in the rows)")
        self.W = W.cuda().contiguous()
        self.home = self.W.device.index
        self.n, self.M, self.K = n, M // 2 if gated else M, K
        self.gated, self.f32 = gated, int(W.dtype == torch.float32)
        self.ptr = self.W.data_ptr()
        self.epi = epilogue(_lib.DN_GLU, glu=glu) if gated else None

    def plan(self, ids, T):
        """The places of T tokens, ids int32 [T, top]."""
        if ids.dtype != torch.int32 or ids.dim() != 2 or ids.shape[0] != T or not ids.is_contiguous():
            raise ValueError(f"ids must be contiguous int32 [{T}, top], got {ids.dtype} {tuple(ids.shape)}")
        stream = _stream(self.home)
        _here(ids, "ids")
        top = ids.shape[1]
        if T * top < group_from(self.n):
            return Places(ids, self.n)
        buf = torch.empty(_lib.dense().lt_dn_experts_plan_ints(T, top, self.n), dtype=torch.int32, device="cuda")
        _lib.call("lt_dn_experts_plan", ids.data_ptr(), T, top, self.n, buf.data_ptr(), stream)
        return Places(ids, self.n, buf, stream)

    def hidden(self, x, ldx, places, h, ldh):
        """h[t*top + j] = glu of the gate and up rows of place (t, j)'s expert, for the rows of x."""
        if not self.gated:
            raise ValueError("the matrices have no gate and up rows: their products are add_sum's")
        stream = _stream(self.home)
        ws = self._workspace(places, stream, "lt_dn_experts_glu_ws", self.K)
        _lib.call("lt_dn_experts_glu", self.ptr, self.K, x, ldx, h, ldh, self.f32, self.M, self.K, places.ref, ctypes.byref(self.epi),
                  None if ws is None else ws.data_ptr(), stream)

    def add_sum(self, h, ldh, places, w, y, ldy, ls=None):
        """y[t] += ls * sum over j of w[t][j] W h[t*top + j]."""
        if self.gated:
            raise ValueError("the matrices are gate and up rows: their product is hidden's")
        stream = _stream(self.home)
        ws = self._workspace(places, stream, "lt_dn_experts_sum_ws", self.M, self.K)
        _lib.call("lt_dn_experts_sum", self.ptr, self.K, h, ldh, y, ldy, self.f32, self.M, self.K, places.ref, w, ls,
                  None if ws is None else ws.data_ptr(), stream)

    def _workspace(self, places, stream, query, *sizes):
        if places.n != self.n:
            raise ValueError(f"places of {places.n} experts, the matrices are of {self.n}")
        if places.stream is not None and places.stream != stream:        # the order's memory is ours to keep until this stream has read it
            places.buf.record_stream(torch.cuda.current_stream())
        n = 0 if places.buf is None else getattr(_lib.dense(), query)(places.T, places.top, *sizes, self.f32)
        return torch.empty(n, dtype=torch.float32, device="cuda") if n else None


# --------------------------------------------------------------------------- delta rule

def delta_chunked_from(ctas):
    """Tokens of the longest sequence from which on bf16 rows are walked in chunks, and not in token order, which takes no
    preparation but more per token, the more CTAs (of 16 value columns) share one of the 148 SMs.  (us in token order / in chunks: 16 heads of
    128, 128 CTAs: 256 tokens 35 / 37, 384 51 / 41; 32 heads: 128 tokens 29 / 36, 176 38 / 39, 256 54 / 42; four sequences of 16 heads: 64 tokens
    31 / 36, 96 43 / 43, 128 55 / 43.  The limits are those of heads of 128; smaller ones meet later, larger ones sooner: 28 heads of 64 256 tokens 28 / 29,
    64 of them 176 tokens 29 / 34 and 256 40 / 36, four sequences of 28 96 tokens 31 / 37 and 128 40 / 37; 8 heads of 256 176 tokens 53 / 53, 16 of
    them 96 tokens 60 / 57 and 176 105 / 62.)"""
    return DELTA_CHUNKED_FROM if DELTA_CHUNKED_FROM is not None else 256 if ctas <= 148 else 176 if ctas <= 296 else 96


DELTA_CHUNKED_FROM = None       # a number: whatever the sizes
DELTA_PORTION = 4096            # rows of a sequence that are walked in chunks at a time, at most (a multiple of 64)
# fp32 elements of workspace that the chunks of all sequences in a walk take together, or one chunk of each: 1 GB.  (us with 512 MB / 1 GB / 2 GB /
# all at once: eight sequences of 4096 rows, 32 heads of 128 3417 / 3281 / 3213 / 3168; of 2048 rows, 16 heads 878 / 840 / 841 / 840; one of 4096
# rows, 16 heads of 256 x 512 1383 / 1308 / 1236 / 1236.)
DELTA_WORKSPACE = 1 << 28


class DeltaRule:
    """Gated delta rule of H heads on G key heads: rows() over the rows of sequences, step() for one token with its convolution
    (taps, conv, conv_b, dt_bias and A as in lt_dn_delta, on the device).  dim and vdim are the padded sizes."""

    def __init__(self, H, G, dim, vdim, dtype, q_scale, eps, taps=0, conv=None, conv_b=None, dt_bias=None, A=None):
        if H % G or dim % 8 or vdim % 8:
            raise ValueError(f"{H} heads on {G} key heads, sizes {dim} and {vdim} (multiples of 8)")
        if dtype not in DTYPES.values():
            raise ValueError(f"rows of {dtype}")
        self.H, self.G, self.dim, self.vdim = H, G, dim, vdim
        self.f32 = int(dtype == torch.float32)
        C = H * vdim + 2 * G * dim
        for name, t, shape in (("conv", conv, (taps, C)), ("conv_b", conv_b, (C,)), ("dt_bias", dt_bias, (H,)), ("A", A, (H,))):
            if t is not None and tuple(t.shape) != shape:        # a token's step reads all of it
                raise ValueError(f"{name} {tuple(t.shape)} for {taps} taps, {C} channels and {H} heads")
        self.keep = [None if t is None else t.float().contiguous() for t in (conv, conv_b, dt_bias, A)]
        self.home = next((t.device.index for t in self.keep if t is not None), None)
        self.desc = _lib.DnDelta(H, G, dim, vdim, float(q_scale), float(eps), taps, *[None if t is None else _here(t, "a constant").data_ptr()
                                                                                   for t in self.keep])
        self._ref = ctypes.byref(self.desc)
        one = _lib.DnSeqs(n=1)
        one.rows[0], one.S[0] = 1, 16            # the size of one chunk's workspace; nothing is read
        self.chunk = _lib.dense().lt_dn_delta_chunked_ws(self._ref, ctypes.byref(one))

    def rows(self, q, k, v, ld, la, beta, ldh, o, ldo, states, rows, ldb=None):
        """Consecutive rows of sequences: rows[i] of them with the state at states[i], from row 0 on.  la and beta have row stride
        ldh, or beta ldb of its own."""
        ldb = ldh if ldb is None else ldb
        if len(states) != len(rows):
            raise ValueError(f"{len(states)} states for {len(rows)} sequences")
        if len(set(states)) != len(states):
            raise ValueError("two sequences with one state")
        if any(r < 0 for r in rows):
            raise ValueError(f"rows of sequences {rows}")
        at, stream = 0, _stream(self.home)
        for i in range(0, len(rows), _lib.DN_SEQS):
            part = rows[i:i + _lib.DN_SEQS]
            seqs = _lib.DnSeqs(n=len(part))
            for j, r in enumerate(part):
                seqs.start[j], seqs.rows[j], seqs.S[j] = at, r, states[i + j]
                at += r
            args = (q, k, v, ld, la, ldh, beta, ldb, o, ldo)
            ctas = (self.vdim + 15) // 16 * self.H * len(part)
            if self.f32 or max(part) < delta_chunked_from(ctas) or self.dim > 256 or self.vdim > 512:
                _lib.call("lt_dn_delta_rows", *args, self.f32, self._ref, ctypes.byref(seqs), stream)
                continue
            starts, done = seqs.start[:len(part)], 0
            while done < max(part):
                left = sum(r > done for r in part)
                portion = min(DELTA_PORTION, 64 * max(1, DELTA_WORKSPACE // max(1, self.chunk * left)))
                for j, r in enumerate(part):
                    seqs.start[j], seqs.rows[j] = starts[j] + min(done, r), max(0, min(r - done, portion))
                done += portion
                ws = torch.empty(_lib.dense().lt_dn_delta_chunked_ws(self._ref, ctypes.byref(seqs)), dtype=torch.float32, device="cuda")
                _lib.call("lt_dn_delta_chunked", *args, self._ref, ctypes.byref(seqs), ws.data_ptr(), stream)
                del ws           # ahead of the next portion's, which takes its place

    def step(self, row, dt, beta, ring, S, o, len_, ticket):
        _lib.call("lt_dn_delta_step", row, dt, beta, ring, S, o, self.f32, len_, ticket, self._ref, _stream(self.home))
