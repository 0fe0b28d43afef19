"""Host-side plans behind the generated modules' `forward`.

A plan fixes the parameters of one computation (taken from the IR and the
tensor-metadata constants), owns the scratch buffers the HIP library needs
beyond the caller's tensors, and calls the C ABI on torch's current stream.
Scratch is allocated on the first call only (the reference's drivers always
run warm-up calls before capturing a graph, convert_eval_rms.py:253-263), so
`forward` allocates nothing afterwards and is safe under graph capture.
Such a plan serves one call at a time (CachedAttention, CachedAttentionPlan and
what stands behind them below may be shared by threads and streams).

Reference semantics (baseline/ref_rms.py:28-403) are the defaults: no softmax
scale, no causal mask, as many KV heads as query heads, RMSNorm without eps
or weight, KeyFormer temperature 1.5 with the noise passed as a tensor.  The
benchmark configurations override them through the constructor.
"""
import torch

from . import ext


def _f32_view(t, rows, cols, cache, key):
    """fp32 [rows, cols] buffer for the kernels; returns (buffer, needs_copy_back)."""
    if t.dtype == torch.float32:
        return t, False
    buf = cache.get(key)
    if buf is None or buf.shape != (rows, cols) or buf.device != t.device:
        buf = torch.empty(rows, cols, dtype=torch.float32, device=t.device)
        cache[key] = buf
    return buf, True


class AttentionPlan:
    """QKV projection + KV-cache append + attention (vanilla | keyformer | roco),
    optionally with PreNorm and/or QKNorm."""

    def __init__(self, variant="vanilla", M=None, N=None, D=None, H=None, P=0, prenorm=False, qknorm=False, tau=1.5,
                 scale=1.0, causal=False, n_kv_heads=None, eps=0.0, noise_seed=0, as_mean_var=False):
        if variant not in ("vanilla", "keyformer", "roco"):
            raise ValueError("unknown attention variant %r" % variant)
        self.variant, self.M, self.N, self.D, self.H, self.P = variant, M, N, D, H, P
        self.prenorm, self.qknorm, self.tau = prenorm, qknorm, tau
        self.scale, self.causal, self.n_kv_heads, self.eps = scale, causal, n_kv_heads, eps
        self.noise_seed, self.as_mean_var = noise_seed, as_mean_var
        self._cache = {}
        self._last = None

    def _params(self, X, WK):
        """Parameters and scratch size of a call; the last ones are kept, since most callers repeat a shape (filling the
        structure and asking for the size take 8 us, as long as a kernel of a decode step)."""
        S, N = X.shape
        if self.M is not None and S != self.M:
            raise ValueError("X has %d rows, the plan was built for M = %d" % (S, self.M))
        kv_cols = WK.shape[1]
        key = (S, N, kv_cols, self.D, self.H, self.n_kv_heads, self.P, self.scale, self.causal, self.eps, self.prenorm,
               self.qknorm, self.tau, self.noise_seed)
        last = self._last
        if last is None or last[0] != key:
            H = self.H if self.H is not None else N // self.D
            Hkv = self.n_kv_heads if self.n_kv_heads is not None else kv_cols // self.D
            p = ext.attn_params(H, Hkv, self.D, S, kv_prefix=self.P, scale=self.scale, causal=self.causal,
                                rms_eps=self.eps, prenorm=self.prenorm, qknorm=self.qknorm, tau=self.tau,
                                noise_seed=self.noise_seed)
            self._last = last = (key, p, ext.qkv_scratch_bytes(p, N), H)
        return last[1], last[2], S, last[3]

    def _scratch(self, need, X):
        buf = self._cache.get("scratch")
        if buf is None or buf.numel() < need or buf.device != X.device:
            buf = torch.empty(need, dtype=torch.uint8, device=X.device)
            self._cache["scratch"] = buf
        return buf

    def run(self, X, WQ, WK, WV, O2, K_cache=None, V_cache=None, noise=None, C_out=None, C_out1=None, C_out2=None,
            norm_w=None, lse=None):
        p, need, S, H = self._params(X, WK)
        scratch = self._scratch(need, X)
        L = self.P + S
        if self.variant == "vanilla":
            ext.qkv_attention(X, norm_w, WQ, WK, WV, K_cache, V_cache, scratch, lse, O2, p)
        elif self.variant == "keyformer":
            if C_out is None:
                raise ValueError("keyformer needs the C_out buffer")
            score, back = _f32_view(C_out, H, L, self._cache, "score")
            ext.keyformer(X, norm_w, WQ, WK, WV, K_cache, V_cache, scratch, noise, O2, score, p)
            if back:
                C_out.copy_(score)
        else:
            if C_out1 is None or C_out2 is None:
                raise ValueError("roco needs the C_out1 and C_out2 buffers")
            s1, b1 = _f32_view(C_out1, H, L, self._cache, "s1")
            s2, b2 = _f32_view(C_out2, H, L, self._cache, "s2")
            ext.roco(X, norm_w, WQ, WK, WV, K_cache, V_cache, scratch, O2, s1, s2, p, as_mean_var=self.as_mean_var)
            if b1:
                C_out1.copy_(s1)
            if b2:
                C_out2.copy_(s2)


class CachedAttention:
    """Caches of several sequences of different lengths, in 16 or in 4 bits, and attention over them: new rows are written
    (`append`), rows read back (`read`), and tokens attend to what their sequence holds (`attend`), all of it or, with
    `window`, its last `window` keys and its first `sinks`.

    Caches are [batch, KV heads, rows, head_dim], or `make_cache`'s 4-bit pair of codes and scales.  `lens` (int32 on the
    device, None: all `kv_len`) holds the lengths with the call's tokens, which are the last ones of each sequence; a sequence
    with fewer has its first rows as padding.  `kv_len` (None: all rows of the cache) bounds the lengths.

    An object keeps a scratch buffer for every stream it attends on; a call under graph capture takes one of the graph's own, so
    that graphs share none, and calls of several threads on one stream take one each."""

    def __init__(self, n_q_heads, n_kv_heads, head_dim, scale=None, causal=True, window=0, sinks=0):
        self.head_dim = head_dim
        # (the sizes of a call are read off its tensors)
        self._p = ext.cache_params(0, n_kv_heads, head_dim, 0, 0, n_q_heads=n_q_heads, scale=scale, causal=causal, window=window,
                                   sinks=sinks)
        ext.native()  # (loaded now, not by a call under capture)
        self._scratch = {}

    def __getstate__(self):
        """Copies start without scratch (and a module cannot be copied: the binding is looked up by each call)."""
        return dict(self.__dict__, _scratch={})

    @staticmethod
    def make_cache(batch, n_kv_heads, rows, head_dim, device):
        """Codes and scales of one 4-bit cache (one for keys, one for values)."""
        return (torch.zeros(batch, n_kv_heads, rows, head_dim // 2, dtype=torch.uint8, device=device),
                torch.ones(batch, n_kv_heads, rows, head_dim // 32, dtype=torch.uint8, device=device))

    def append(self, K, V, k_cache, v_cache, k_scales=None, v_scales=None, lens=None, kv_len=None):
        """K, V [batch * tokens, KV heads * head_dim] to the last rows of their sequences."""
        st = ext.native().cache_append_rows(K, V, k_cache, k_scales, v_cache, v_scales, lens, kv_len, self._p, ext._stream_or_none(K))
        if st:
            ext._check("tri_cache_append", st)

    def read(self, k_cache, v_cache, k_scales=None, v_scales=None, dtype=None, rows=None, lens=None, kv_len=None):
        """The last `rows` rows of every sequence (None: `kv_len`) as k, v [batch, KV heads, rows, head_dim]; zeros where a
        sequence has fewer.  From 4 bits in float16 (None) or bfloat16.  k and v are the halves of one allocation: what keeps one
        keeps the memory of both (`clone` for one alone, also to save it)."""
        if k_scales is None:
            if dtype is not None and dtype != k_cache.dtype:
                raise ValueError("rows of a 16-bit cache are read as they are, %s" % k_cache.dtype)
            dtype = k_cache.dtype
        elif dtype not in (None, torch.float16, torch.bfloat16):
            raise ValueError("rows are read as float16 or bfloat16")
        r = ext.native().cache_read_rows(k_cache, k_scales, v_cache, v_scales, lens, rows, dtype is torch.bfloat16, kv_len,
                                         self._p, ext._stream_or_none(k_cache))
        if type(r) is int:
            ext._check("tri_cache_read", r)
        return r

    def attend(self, Q, k_cache, v_cache, k_scales=None, v_scales=None, lens=None, kv_len=None, out=None, want_lse=False):
        """Q [batch * tokens, query heads * head_dim] over the caches, which hold the tokens' own keys already.  Returns
        the output like Q, and with `want_lse` the log-sum-exp [batch, query heads, tokens] beside it."""
        stream = ext._stream_or_none(Q)
        # The buffer leaves the object for the time of a call: its two launches (parts of the keys, their merge) are enqueued
        # without the interpreter lock, and another thread's call on the stream, which may enqueue its own between them, finds none.
        kept = self._scratch.pop(stream, None)
        capturing = kept is not None and torch.cuda.is_current_stream_capturing()
        call = ext.native().cache_attend
        r = call(Q, k_cache, k_scales, v_cache, v_scales, lens, None if capturing else kept, out, want_lse, kv_len, self._p, stream)
        if type(r) is int and r > 0:  # bytes of scratch: the first call of its size, or a captured one
            scratch = torch.empty(r, dtype=torch.uint8, device=Q.device)
            if not torch.cuda.is_current_stream_capturing():
                kept = scratch
            r = call(Q, k_cache, k_scales, v_cache, v_scales, lens, scratch, out, want_lse, kv_len, self._p, stream)
        if kept is not None:
            self._scratch[stream] = kept
        if type(r) is int:
            ext._check("tri_cache_attention", r)
        return r


class CachedAttentionPlan:
    """AttentionPlan's block - [PreNorm,] Q/K/V projection, [QKNorm,] append, attention - for the next tokens of several
    sequences over the caches of `CachedAttention`: X [batch * tokens, N], and what its methods take.  A call's buffers come
    from the allocator: prompts, single tokens and captured graphs of one plan share none."""

    def __init__(self, n_q_heads, n_kv_heads, head_dim, scale=None, causal=True, window=0, sinks=0, prenorm=False, qknorm=False,
                 eps=0.0):
        self.attention = CachedAttention(n_q_heads, n_kv_heads, head_dim, scale=scale, causal=causal, window=window, sinks=sinks)
        self.prenorm, self.qknorm, self.eps = prenorm, qknorm, eps

    def _project(self, X, W, norm):
        rows, cols = X.shape[0], W.shape[1]
        need = ext.gemm_workspace_bytes(rows, X.shape[1], cols)
        y = X.new_empty(rows, cols)
        ext.matmul(X, W, None, y, X.new_empty(need, dtype=torch.uint8) if need else None)
        if not norm:
            return y
        D = self.attention.head_dim
        z = torch.empty_like(y)
        ext.rmsnorm(y.view(-1, D), None, z.view(-1, D), self.eps)
        return z

    def run(self, X, WQ, WK, WV, O2, k_cache, v_cache, k_scales=None, v_scales=None, lens=None, kv_len=None, norm_w=None,
            want_lse=False):
        if norm_w is not None and not self.prenorm:
            raise ValueError("a norm weight without PreNorm")
        # (the products and norms launch on the current GPU, and would read another's memory, or the host's, as if it were its own)
        if not X.is_cuda or any(t is not None and t.device != X.device for t in (WQ, WK, WV, norm_w)):
            raise ValueError("the tensors of a call have to be on one GPU")
        if X.device.index != torch.cuda.current_device():
            with torch.cuda.device(X.device):
                return self.run(X, WQ, WK, WV, O2, k_cache, v_cache, k_scales, v_scales, lens, kv_len, norm_w, want_lse)
        if self.prenorm:
            xn = X.new_empty(X.shape)
            ext.rmsnorm(X, norm_w, xn, self.eps)
            X = xn
        K = self._project(X, WK, self.qknorm)
        V = self._project(X, WV, False)
        self.attention.append(K, V, k_cache, v_cache, k_scales, v_scales, lens=lens, kv_len=kv_len)
        Q = self._project(X, WQ, self.qknorm)
        return self.attention.attend(Q, k_cache, v_cache, k_scales, v_scales, lens=lens, kv_len=kv_len, out=O2, want_lse=want_lse)


class FfnBlockPlan:
    """The reference-shaped FFN block: output projection + residual + RMSNorm +
    SwiGLU + down projection (+ residual + RMSNorm with `falcon_tail`)."""

    def __init__(self, falcon_tail=False):
        self.falcon_tail = falcon_tail
        self._cache = {}

    def _buf(self, key, given, shape, dtype, dev):
        if given is not None:
            return given
        b = self._cache.get(key)
        if b is None or tuple(b.shape) != tuple(shape) or b.device != dev:
            b = torch.empty(*shape, dtype=dtype, device=dev)
            self._cache[key] = b
        return b

    def run(self, O2, WO, X, WFF1a, WFF1b, WFF2, attn_O2=None, FF1=None, FF2=None, O_FF_norm=None):
        M, N = O2.shape
        F = WFF1a.shape[1]
        dev = O2.device
        attn = self._buf("attn", attn_O2, (M, N), torch.float16, dev)
        ff1 = self._buf("ff1", FF1, (M, F), torch.float16, dev)
        ff2 = self._buf("ff2", FF2, (M, N), torch.float16, dev)
        rows = self._buf("rows", None, (M,), torch.float32, dev)
        if self.falcon_tail and O_FF_norm is None:
            raise ValueError("the Falcon-shaped block needs the O_FF_norm buffer")
        ws_bytes = ext.ffn_workspace_bytes(M, N, F)  # non-zero for few rows (the reference's M = 16)
        ws = self._buf("ws", None, (ws_bytes,), torch.uint8, dev) if ws_bytes else None
        ext.ffn_block(O2, WO, X, WFF1a, WFF1b, WFF2, attn, rows, ff1, ff2, O_FF_norm if self.falcon_tail else None,
                      workspace=ws)


class RmsNormPlan:
    """Standalone RMSNorm (reference point: no eps, no weight)."""

    def __init__(self, eps=0.0):
        self.eps = eps

    def run(self, O_FF, O_FF_norm, weight=None):
        ext.rmsnorm(O_FF, weight, O_FF_norm, self.eps)


class FfnPlan:
    """The benchmark configuration's plain FFNs: SwiGLU (gate, up, down) or
    GELU (w1, w2).  The hidden activation is plan-owned scratch."""

    def __init__(self, activation="swiglu"):
        if activation not in ("swiglu", "gelu"):
            raise ValueError("activation must be swiglu or gelu")
        self.activation = activation
        self._hidden = None
        self._ws = None

    def run(self, X, W1, W2, out, W_up=None):
        T, F = X.shape[0], W1.shape[1]
        if self._hidden is None or tuple(self._hidden.shape) != (T, F) or self._hidden.device != X.device:
            self._hidden = torch.empty(T, F, dtype=torch.float16, device=X.device)
        ws_bytes = ext.ffn_workspace_bytes(T, X.shape[1], F)
        if ws_bytes and (self._ws is None or self._ws.numel() < ws_bytes or self._ws.device != X.device):
            self._ws = torch.empty(ws_bytes, dtype=torch.uint8, device=X.device)
        ws = self._ws if ws_bytes else None
        if self.activation == "swiglu":
            if W_up is None:
                raise ValueError("SwiGLU needs W_up")
            ext.ffn_swiglu(X, W1, W_up, W2, self._hidden, out, workspace=ws)
        else:
            ext.ffn_gelu(X, W1, W2, self._hidden, out, workspace=ws)


class Fp4Matmul:
    """Products over weights in 4 bits: y = x . w^T, w as `quantize` makes it of an [N, K] matrix (torch.nn.Linear's layout) -
    codes [N, K / 2] and scales [N, K / 32]; with `quantize_x`, x goes to 4 bits as well, and the product runs on the 4-bit matrix
    instructions.  Every call's buffers come from the allocator: an object may be shared by threads, streams and graphs."""

    def __init__(self, quantize_x=False):
        self.quantize_x = bool(quantize_x)
        ext.native()  # (loaded now, not by a call under capture)

    @staticmethod
    def quantize(X):
        """Codes and scales of the rows of X [M, K], K a multiple of 32."""
        r = ext.native().fp4_quantize_new(X, ext._stream_or_none(X))
        if type(r) is int:
            ext._check("tri_fp4_quantize", r)
        return r

    @staticmethod
    def dequantize(codes, scales, dtype=torch.float16):
        """The values that codes and scales stand for, in float16 or bfloat16."""
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("values are float16 or bfloat16")
        r = ext.native().fp4_dequantize_new(codes, scales, dtype is torch.bfloat16, ext._stream_or_none(codes))
        if type(r) is int:
            ext._check("tri_fp4_dequantize", r)
        return r

    def run(self, X, W, w_scales, x_scales=None, out=None, dtype=torch.float16):
        """X [M, K], or its codes with `x_scales` (the result is then of type `dtype`, or `out`'s)."""
        if x_scales is not None and dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("results are float16 or bfloat16")
        r = ext.native().fp4_matmul_new(X, x_scales, W, w_scales, out, self.quantize_x and x_scales is None,
                                        dtype is torch.bfloat16, ext._stream_or_none(X))
        if type(r) is int:
            ext._check("tri_fp4_matmul", r)
        return r


class Router:
    """Experts of every token and their weights from a router's logits: scores are the softmax or sigmoid of the logits, experts
    are chosen by score + bias, `top_k` of them in descending order (ties: the lowest index), out of the `top_groups` best of
    `groups` groups of neighbours - a group counts its `group_top` (1 or 2) largest - and weighted with their scores, over the
    sum of the chosen if `renormalize`, times `scale`.  (One group stays whatever it counts: 1 and 2 are the same there.)"""

    def __init__(self, top_k, scores="softmax", groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0):
        if scores not in ("softmax", "sigmoid"):
            raise ValueError("scores must be softmax or sigmoid")
        if groups == 1 and group_top == 2:
            group_top = 1  # (the entry point has that as the one way to say it)
        self.top_k = top_k
        self._p = ext.route_params(top_k, sigmoid=scores == "sigmoid", groups=groups, top_groups=top_groups, group_top=group_top,
                                   renormalize=renormalize, scale=scale)
        ext.native()

    def route(self, logits, bias=None):
        """logits [T, E], bias float32 [E]: ids int32 [T, top_k] and weights float32 [T, top_k]."""
        r = ext.native().route_new(logits, bias, self._p, ext._stream_or_none(logits))
        if type(r) is int:
            ext._check("tri_route", r)
        return r


class ExpertsFfn:
    """The SwiGLU FFN of the experts that each token chose: out[t] = sum over i of weights[t, i] * FFN_ids[t, i](x[t]).  Weights are
    [E, F, N] (gate, up) and [E, N, F] (down), torch.nn.Linear's layout for each expert, of x's type or in 4 bits (codes, and
    scales of all three, as `Fp4Matmul.quantize` makes them of an expert's matrix).  ids outside [0, E) count nothing.  Every call's
    buffers come from the allocator: an object may be shared by threads, streams and graphs."""

    def __init__(self):
        ext.native()

    def run(self, X, ids, weights, W_gate, W_up, W_down, gate_scales=None, up_scales=None, down_scales=None, out=None):
        r = ext.native().experts_ffn_new(X, ids, weights, W_gate, gate_scales, W_up, up_scales, W_down, down_scales, out,
                                         ext._stream_or_none(X))
        if type(r) is int:
            ext._check("tri_experts_ffn", r)
        return r


class RoutedFfnPlan:
    """The FFN half of a layer with experts: [RMSNorm,] the router's product, routing, and the experts' FFN: X [T, N], W_router
    [N, E] (E a multiple of 8, as the product wants it), and what `Router` and `ExpertsFfn` take.  A call's buffers come from the
    allocator.

    The logits are a result of `ext.matmul`, in X's type as all its results are (summed in fp32): in bfloat16 equal logits are common
    among many experts, and the lowest index wins.  A model that was trained to route on fp32 logits computes those itself and
    calls `Router` and `ExpertsFfn`, which is all that happens here."""

    def __init__(self, top_k, scores="softmax", groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0, prenorm=False,
                 eps=0.0):
        self.router = Router(top_k, scores=scores, groups=groups, top_groups=top_groups, group_top=group_top,
                             renormalize=renormalize, scale=scale)
        self.experts = ExpertsFfn()
        self.prenorm, self.eps = prenorm, eps

    def run(self, X, W_router, W_gate, W_up, W_down, gate_scales=None, up_scales=None, down_scales=None, bias=None, norm_w=None,
            out=None):
        if norm_w is not None and not self.prenorm:
            raise ValueError("a norm weight without PreNorm")
        # (the product and the norm launch on the current GPU, and would read another's memory, or the host's, as if it were its own)
        if not X.is_cuda or any(t is not None and t.device != X.device for t in (W_router, norm_w)):
            raise ValueError("the tensors of a call have to be on one GPU")
        if X.device.index != torch.cuda.current_device():
            with torch.cuda.device(X.device):
                return self.run(X, W_router, W_gate, W_up, W_down, gate_scales, up_scales, down_scales, bias, norm_w, out)
        if self.prenorm:
            xn = X.new_empty(X.shape)
            ext.rmsnorm(X, norm_w, xn, self.eps)
            X = xn
        logits = X.new_empty(X.shape[0], W_router.shape[1])
        need = ext.gemm_workspace_bytes(X.shape[0], X.shape[1], W_router.shape[1])
        ext.matmul(X, W_router, None, logits, X.new_empty(need, dtype=torch.uint8) if need else None)
        ids, weights = self.router.route(logits, bias)
        return self.experts.run(X, ids, weights, W_gate, W_up, W_down, gate_scales, up_scales, down_scales, out=out)
