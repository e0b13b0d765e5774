"""Host-side mirror of the conv section of Dragon-Alpha's CudaFloat32EngineBase.

`CudaFloat32EngineBase` keeps the reference's address-level operator methods (same names, same
argument order, same option setters and the same IllegalArgument checks, raised as ValueError):
src/alpha_src/z/dragon/engine/cuda/CudaFloat32EngineBase.java:1322-2007.  `Engine` adds the
tensor-level calls with the shape inference of src/alpha_src/z/dragon/engine/Engine.java:1541-1829
and the pad-to-4 memory rule of src/alpha_src/z/dragon/engine/Tensor.java:208-221.

PyTorch only provides device memory and streams here; every contraction runs in
libalpha_conv_b200.so.  There is no CPU or PyTorch fallback: a missing library raises ImportError.
"""
import contextlib
import ctypes as C
import functools
import itertools
import operator
import struct

import torch

from . import lib as _l


def _stream(stream=None):
    """The raw handle of `stream`, or of the current device's current stream."""
    if stream is not None:
        return stream.cuda_stream
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


# Shapes as the C structures the library reads (it never writes them): a program calls a few layers over and over.  The caches see
# plain ints only (and the slope as a float): 3.0 would find the entry of 3, and a tensor the entry it made before its value changed.
_cached_conv_shape = functools.lru_cache(maxsize=512)(_l.AlphaConvShape)
_cached_pool_shape = functools.lru_cache(maxsize=512)(_l.AlphaPoolShape)
_cached_fc_shape = functools.lru_cache(maxsize=512)(_l.AlphaFcShape)


def _conv_shape(*dims):
    return _cached_conv_shape(*map(operator.index, dims))


def _pool_shape(*dims):
    return _cached_pool_shape(*map(operator.index, dims))


def _fc_shape(rows, IC, OC, dtype, act, k):
    return _cached_fc_shape(*map(operator.index, (rows, IC, OC, dtype, act)), float(k))


def _new(like, shape, dtype=torch.float32):
    return like.new_empty(shape, dtype=dtype)


class CudaFloat32EngineBase:
    """Address-level operators.  Arguments are device addresses (ints) or torch CUDA tensors."""

    def __init__(self, stream=None, math=None, algo=None):
        """math ('3xtf32' / 'tf32') and algo ('auto' / 'tensor' / 'simt' / 'winograd') are this engine's own
        settings, passed with every call; None follows the process-wide default of lib.set_math_mode /
        lib.set_algo.  Two engines of one process may differ."""
        self._lib = _l.load()
        self._stream = stream
        self._math = -1 if math is None else {"3xtf32": _l.ALPHA_MATH_3XTF32, "tf32": _l.ALPHA_MATH_TF32}[math]
        self._algo = -1 if algo is None else {"auto": 0, "tensor": 1, "simt": 2, "winograd": 3}[algo]
        # Option flags of the reference.  There they choose among SIMT kernel families (texture loads,
        # remoded weights, the V2 tilings, split-K part counts); every family maps onto the same
        # tensor-core kernels here, so the setters below only store the value: they exist so that host
        # code written against the reference's engine runs unchanged, and nothing reads them.
        self._conv3D_useTexture = True
        self._conv3D_remode = True
        self._conv3D_remode_V2_Q = 1.05
        self._conv3D_V2_Q = 1.25
        self._dW_SplitKThreshold = 512
        self._dW_SK_MaxPartNum = 16
        self._dW_SK_V2_Q = 1.15
        self._dX_s1_useTexture = True
        self._dX_ks_useTexture = False
        self._dX_ks_V2_Q = 1.1
        self._dX_s1_V2_Q = 1.1

    # ---- fluent option setters (CudaFloat32EngineBase.java:1324-1352, 1630-1663, 1765-1793) ----
    def conv3D_useTexture(self, flag=None):
        if flag is None:
            return self._conv3D_useTexture
        self._conv3D_useTexture = bool(flag)
        return self

    def conv3D_remode(self, flag=None):
        if flag is None:
            return self._conv3D_remode
        self._conv3D_remode = bool(flag)
        return self

    def conv3D_remode_V2_Q(self, Q=None):
        if Q is None:
            return self._conv3D_remode_V2_Q
        if Q < 1.04999:
            raise ValueError("Q must >= 1.05")
        self._conv3D_remode_V2_Q = float(Q)
        return self

    def conv3D_V2_Q(self, Q=None):
        if Q is None:
            return self._conv3D_V2_Q
        if Q < 1.09999:
            raise ValueError("Q must >= 1.1")
        self._conv3D_V2_Q = float(Q)
        return self

    def dconv3D_deltaW_SplitKThreshold(self, threshold=None):
        if threshold is None:
            return self._dW_SplitKThreshold
        if threshold & (threshold - 1):
            raise ValueError("threshold must be a power of 2")
        if threshold < 256:
            raise ValueError("threshold must >= 256")
        self._dW_SplitKThreshold = int(threshold)
        return self

    def dconv3D_deltaW_SK_MaxPartNum(self, maxPartNum=None):
        if maxPartNum is None:
            return self._dW_SK_MaxPartNum
        if maxPartNum < 4:
            raise ValueError("maxPartNum must >= 4")
        self._dW_SK_MaxPartNum = int(maxPartNum)
        return self

    def dconv3DdeltaW_SK_V2_Q(self, Q=None):
        if Q is None:
            return self._dW_SK_V2_Q
        if Q < 1.1:
            raise ValueError("Q >= 1.1")
        self._dW_SK_V2_Q = float(Q)
        return self

    def dconv3D_deltaX_s1_useTexture(self, flag=None):
        if flag is None:
            return self._dX_s1_useTexture
        self._dX_s1_useTexture = bool(flag)
        return self

    def dconv3D_deltaX_ks_useTexture(self, flag=None):
        if flag is None:
            return self._dX_ks_useTexture
        self._dX_ks_useTexture = bool(flag)
        return self

    # ---- operators ------------------------------------------------------------------------------
    def _own_settings(self):
        return self._math >= 0 or self._algo >= 0

    @staticmethod
    def _addr(a):
        return a.data_ptr() if isinstance(a, torch.Tensor) else int(a)

    @staticmethod
    def _addr_or_none(a):
        return a if a is None or type(a) is int else a.data_ptr() if isinstance(a, torch.Tensor) else int(a)

    def conv3D(self, Y_address, OH, OW, X_address, IH, IW, W_address, FH, FW, N, IC, OC, sh, sw, ph, pw):
        """CudaFloat32EngineBase.conv3D (:1355-1474)."""
        a = self._addr
        if self._own_settings():
            shp = _conv_shape(N, IH, IW, IC, OC, FH, FW, OH, OW, sh, sw, ph, pw)
            return _l.check(self._lib.alpha_conv3d_forward_ex(C.byref(shp), a(X_address), a(W_address), None, a(Y_address),
                                                              self._math, self._algo, _stream(self._stream)))
        _l.check(self._lib.alpha_engine_conv3D(a(Y_address), OH, OW, a(X_address), IH, IW, a(W_address),
                                               FH, FW, N, IC, OC, sh, sw, ph, pw, _stream(self._stream)))

    def conv3D_biased(self, Y_address, OH, OW, X_address, IH, IW, W_address, FH, FW, Bias_address, N, IC,
                      OC, sh, sw, ph, pw):
        """CudaFloat32EngineBase.conv3D_biased (:1478-1627); the bias add is fused in the epilogue."""
        a = self._addr
        if self._own_settings():
            shp = _conv_shape(N, IH, IW, IC, OC, FH, FW, OH, OW, sh, sw, ph, pw)
            return _l.check(self._lib.alpha_conv3d_forward_ex(C.byref(shp), a(X_address), a(W_address), a(Bias_address),
                                                              a(Y_address), self._math, self._algo, _stream(self._stream)))
        _l.check(self._lib.alpha_engine_conv3D_biased(a(Y_address), OH, OW, a(X_address), IH, IW,
                                                      a(W_address), FH, FW, a(Bias_address), N, IC, OC,
                                                      sh, sw, ph, pw, _stream(self._stream)))

    def dconv3D_deltaW(self, deltaW_address, FH, FW, X_address, IH, IW, deltaY_address, OH, OW, N, IC, OC,
                       sh, sw, ph, pw):
        """CudaFloat32EngineBase.dconv3D_deltaW (:1666-1762)."""
        a = self._addr
        if self._own_settings():
            shp = _conv_shape(N, IH, IW, IC, OC, FH, FW, OH, OW, sh, sw, ph, pw)
            return _l.check(self._lib.alpha_conv3d_deltaW_ex(C.byref(shp), a(X_address), a(deltaY_address), a(deltaW_address),
                                                             self._math, self._algo, _stream(self._stream)))
        _l.check(self._lib.alpha_engine_dconv3D_deltaW(a(deltaW_address), FH, FW, a(X_address), IH, IW,
                                                       a(deltaY_address), OH, OW, N, IC, OC, sh, sw, ph,
                                                       pw, _stream(self._stream)))

    def dconv3D_deltaX(self, deltaX_address, IH, IW, deltaY_address, OH, OW, W_address, FH, FW, N, IC, OC,
                       sh, sw, ph, pw):
        """CudaFloat32EngineBase.dconv3D_deltaX (:1796-2005)."""
        a = self._addr
        if self._own_settings():
            shp = _conv_shape(N, IH, IW, IC, OC, FH, FW, OH, OW, sh, sw, ph, pw)
            return _l.check(self._lib.alpha_conv3d_deltaX_ex(C.byref(shp), a(deltaY_address), a(W_address), a(deltaX_address),
                                                             self._math, self._algo, _stream(self._stream)))
        _l.check(self._lib.alpha_engine_dconv3D_deltaX(a(deltaX_address), IH, IW, a(deltaY_address), OH,
                                                       OW, a(W_address), FH, FW, N, IC, OC, sh, sw, ph,
                                                       pw, _stream(self._stream)))


    # ---- weight-side transforms in caller-owned memory --------------------------------------------------
    def prepare_weights(self, op, W_address, FH, FW, N, IH, IW, OH, OW, IC, OC, sh, sw, ph, pw, stream=None):
        """Enqueues the transform of W that `op` ('forward' / 'deltaX') needs for this layer on `stream` and returns
        the block (a torch uint8 tensor, or None when the operator needs none).  A training loop runs these for
        all layers on a side stream after the optimizer step; conv3D / dconv3D_deltaX then take the block through
        their `prepared` argument.  The caller orders prepare before use."""
        shp = _conv_shape(N, IH, IW, IC, OC, FH, FW, OH, OW, sh, sw, ph, pw)
        nbytes = _l.prepared_weights_bytes(shp, op)
        if nbytes == 0:
            return None
        W = W_address if isinstance(W_address, torch.Tensor) else None
        block = torch.empty(nbytes, dtype=torch.uint8, device=W.device if W is not None else "cuda")
        self.prepare_weights_into(block, op, W_address, FH, FW, N, IH, IW, OH, OW, IC, OC, sh, sw, ph, pw, stream)
        return block

    def prepare_weights_into(self, block, op, W_address, FH, FW, N, IH, IW, OH, OW, IC, OC, sh, sw, ph, pw, stream=None):
        shp = _conv_shape(N, IH, IW, IC, OC, FH, FW, OH, OW, sh, sw, ph, pw)
        _l.check(self._lib.alpha_conv_prepare_weights(C.byref(shp), _l.OPS[op], self._addr(W_address), self._addr(block),
                                                      block.numel(), _stream(stream if stream is not None else self._stream)))

    def conv3D_prepared(self, Y_address, OH, OW, X_address, IH, IW, W_address, FH, FW, N, IC, OC, sh, sw, ph, pw, prepared):
        a = self._addr
        shp = _conv_shape(N, IH, IW, IC, OC, FH, FW, OH, OW, sh, sw, ph, pw)
        _l.check(self._lib.alpha_conv3d_forward_prepared(C.byref(shp), a(X_address), a(W_address),
                                                         a(prepared) if prepared is not None else None,
                                                         prepared.numel() if prepared is not None else 0, None, a(Y_address),
                                                         _stream(self._stream)))

    def dconv3D_deltaX_prepared(self, deltaX_address, IH, IW, deltaY_address, OH, OW, W_address, FH, FW, N, IC, OC, sh, sw, ph, pw,
                                prepared):
        a = self._addr
        shp = _conv_shape(N, IH, IW, IC, OC, FH, FW, OH, OW, sh, sw, ph, pw)
        _l.check(self._lib.alpha_conv3d_deltaX_prepared(C.byref(shp), a(deltaY_address), a(W_address),
                                                        a(prepared) if prepared is not None else None,
                                                        prepared.numel() if prepared is not None else 0, a(deltaX_address),
                                                        _stream(self._stream)))

    # ---- matrix products (CudaFloat32EngineBase.java:1129-1245) ---------------------------------------
    def _mm(self, fn, *args):
        old = self._lib.alpha_conv_get_math_mode() if self._math >= 0 else self._math
        if self._math != old:
            _l.check(self._lib.alpha_conv_set_math_mode(self._math))
            try:
                _l.check(fn(*args))
            finally:
                self._lib.alpha_conv_set_math_mode(old)
        else:
            _l.check(fn(*args))

    def matMul(self, C_address, A_address, B_address, N, M, K):
        """C[N,M] = A[N,K] * B[K,M] (CudaFloat32EngineBase.matMul, :1129-1139)."""
        a = self._addr
        self._mm(self._lib.alpha_engine_matMul, a(C_address), a(A_address), a(B_address), N, M, K, _stream(self._stream))

    def matMul_biased(self, C_address, A_address, B_address, N, M, K, Bias_address):
        """C = A * B + Bias per row (CudaFloat32EngineBase.matMul_biased, :1142-1168)."""
        a = self._addr
        self._mm(self._lib.alpha_engine_matMul_biased, a(C_address), a(A_address), a(B_address), N, M, K, a(Bias_address),
                 _stream(self._stream))

    def matMulT1(self, C_address, A_address, B_address, N, M, K):
        """C[N,M] = A[K,N]^T * B[K,M] (CudaFloat32EngineBase.matMulT1, :1185-1230)."""
        a = self._addr
        self._mm(self._lib.alpha_engine_matMulT1, a(C_address), a(A_address), a(B_address), N, M, K, _stream(self._stream))

    def matMulT2(self, C_address, A_address, B_address, N, M, K):
        """C[N,M] = A[N,K] * B[M,K]^T (CudaFloat32EngineBase.matMulT2, :1233-1245)."""
        a = self._addr
        self._mm(self._lib.alpha_engine_matMulT2, a(C_address), a(A_address), a(B_address), N, M, K, _stream(self._stream))

    def batchMatMul(self, C_address, A_address, B_address, Batch, N, M, BK, AK):
        """C[b] = A[b][N, AK](:, :BK) * B[b][BK, M] (CudaFloat32EngineBase.batchMatMul, :1256-1272)."""
        a = self._addr
        self._mm(self._lib.alpha_engine_batchMatMul, a(C_address), a(A_address), a(B_address), Batch, N, M, BK, AK,
                 _stream(self._stream))

    def batchMatMulT1(self, C_address, A_address, B_address, Batch, CN, AN, M, K):
        """C[b][CN, M] = (A[b][K, AN](:, :CN))^T * B[b][K, M] (CudaFloat32EngineBase.batchMatMulT1, :1277-1287)."""
        a = self._addr
        self._mm(self._lib.alpha_engine_batchMatMulT1, a(C_address), a(A_address), a(B_address), Batch, CN, AN, M, K,
                 _stream(self._stream))

    def batchMatMulT2(self, C_address, A_address, B_address, Batch, N, CM, BM, K):
        """C[b][N, CM](:, :BM) = A[b][N, K] * B[b][BM, K]^T (CudaFloat32EngineBase.batchMatMulT2, :1298-1318)."""
        a = self._addr
        self._mm(self._lib.alpha_engine_batchMatMulT2, a(C_address), a(A_address), a(B_address), Batch, N, CM, BM, K,
                 _stream(self._stream))

    # ---- FullConnect layers of a transformer (no counterpart in the reference, which runs matMul, linear_dual2D_row and the
    # activation one after the other) ----
    def fullConnect(self, Y_address, X_address, W_address, rows, IC, OC, dtype, act, k, Bias_address=None, Residual_address=None, Z_address=None):
        """Y = act(X W^T + Bias) + Residual, Z = X W^T + Bias; addresses of X[rows, IC], W[OC, IC], and so on (alpha_fullConnect)."""
        a = self._addr_or_none
        _l.check(self._lib.alpha_fullConnect(C.byref(_fc_shape(rows, IC, OC, dtype, act, k)), a(X_address), a(W_address), a(Bias_address), a(Residual_address),
                                             a(Z_address), a(Y_address), _stream(self._stream)))

    def fullConnect_glu(self, Y_address, X_address, W_address, rows, IC, OC, dtype, act, k, Bias_address=None, Z_address=None):
        """Y = act(Z[:, :OC]) * Z[:, OC:], Z = X W^T + Bias with W[2 OC, IC] (alpha_fullConnect_glu)."""
        a = self._addr_or_none
        _l.check(self._lib.alpha_fullConnect_glu(C.byref(_fc_shape(rows, IC, OC, dtype, act, k)), a(X_address), a(W_address), a(Bias_address), a(Z_address),
                                                 a(Y_address), _stream(self._stream)))

    def fullConnect_delta(self, deltaX_address, deltaW_address, deltaB_address, deltaY_address, X_address, W_address, Z_address, deltaZ_address, rows, IC, OC,
                          dtype, act, k, glu=False):
        """The gradients of fullConnect, or of fullConnect_glu (alpha_fullConnect_delta, alpha_fullConnect_glu_delta)."""
        a = self._addr_or_none
        fn = self._lib.alpha_fullConnect_glu_delta if glu else self._lib.alpha_fullConnect_delta
        _l.check(fn(C.byref(_fc_shape(rows, IC, OC, dtype, act, k)), a(deltaY_address), a(X_address), a(W_address), a(Z_address), a(deltaZ_address),
                    a(deltaX_address), a(deltaW_address), a(deltaB_address), _stream(self._stream)))

    def fullConnect_softmax_crossEntropy(self, loss_address, lse_address, X_address, W_address, Bias_address, label_address, label_bytes, rows, IC, OC, dtype):
        """loss = lse - z[label], lse = log sum exp z, z = X W^T + Bias (alpha_fullConnect_softmax_crossEntropy)."""
        a = self._addr_or_none
        _l.check(self._lib.alpha_fullConnect_softmax_crossEntropy(C.byref(_fc_shape(rows, IC, OC, dtype, 0, 0.0)), a(X_address), a(W_address), a(Bias_address), a(label_address),
                                                                  label_bytes, a(loss_address), a(lse_address), _stream(self._stream)))

    def fullConnect_softmax_crossEntropy_delta(self, deltaX_address, deltaW_address, deltaB_address, deltaL_address, deltaL_step, X_address, W_address, Bias_address, label_address,
                                               label_bytes, lse_address, rows, IC, OC, dtype):
        """The gradients of fullConnect_softmax_crossEntropy (alpha_fullConnect_softmax_crossEntropy_delta)."""
        a = self._addr_or_none
        _l.check(self._lib.alpha_fullConnect_softmax_crossEntropy_delta(C.byref(_fc_shape(rows, IC, OC, dtype, 0, 0.0)), a(deltaL_address), deltaL_step, a(X_address), a(W_address),
                                                                        a(Bias_address), a(label_address), label_bytes, a(lse_address), a(deltaX_address), a(deltaW_address),
                                                                        a(deltaB_address), _stream(self._stream)))

    # ---- group normalisation (shape: AlphaNormShape) ----
    def groupNorm(self, shape, X_address, gamma_address, beta_address, mean_address, rstd_address, Y_address):
        b, a = self._addr_or_none, self._addr
        _l.check(self._lib.alpha_groupNorm(C.byref(shape), a(X_address), b(gamma_address), b(beta_address), b(mean_address), b(rstd_address), a(Y_address), _stream(self._stream)))
        return self

    def groupNorm_delta(self, shape, deltaY_address, X_address, mean_address, rstd_address, gamma_address, beta_address, deltaX_address, deltaGamma_address, deltaBeta_address):
        b, a = self._addr_or_none, self._addr
        _l.check(self._lib.alpha_groupNorm_delta(C.byref(shape), a(deltaY_address), a(X_address), a(mean_address), a(rstd_address), b(gamma_address), b(beta_address),
                                                 a(deltaX_address), b(deltaGamma_address), b(deltaBeta_address), _stream(self._stream)))
        return self

    # ---- pooling, Java argument order (CudaFloat32EngineBase.java:2012-2215) ----
    def _pool(self, fn, N, IH, IW, IC, FH, FW, OH, OW, sh, sw, ph, pw, *ptrs_and_flags):
        s = _pool_shape(N, IH, IW, IC, FH, FW, OH, OW, sh, sw, ph, pw)
        _l.check(fn(C.byref(s), *ptrs_and_flags, _stream(self._stream)))

    def pool2D_max(self, Y_address, OH, OW, X_address, IH, IW, FH, FW, N, IC, sh, sw, ph, pw):
        a = self._addr
        self._pool(self._lib.alpha_pool2D_max, N, IH, IW, IC, FH, FW, OH, OW, sh, sw, ph, pw, a(X_address), a(Y_address))

    def pool2D_max_indexed(self, Y_address, Index_address, OH, OW, X_address, IH, IW, FH, FW, N, IC, sh, sw, ph, pw):
        a = self._addr
        self._pool(self._lib.alpha_pool2D_max_indexed, N, IH, IW, IC, FH, FW, OH, OW, sh, sw, ph, pw, a(X_address), a(Y_address),
                   a(Index_address))

    def pool2D_avg(self, Y_address, OH, OW, X_address, IH, IW, FH, FW, N, IC, sh, sw, ph, pw):
        a = self._addr
        self._pool(self._lib.alpha_pool2D_avg, N, IH, IW, IC, FH, FW, OH, OW, sh, sw, ph, pw, a(X_address), a(Y_address), 0)

    def pool2D_avg_ignore_padding(self, Y_address, OH, OW, X_address, IH, IW, FH, FW, N, IC, sh, sw, ph, pw):
        a = self._addr
        self._pool(self._lib.alpha_pool2D_avg, N, IH, IW, IC, FH, FW, OH, OW, sh, sw, ph, pw, a(X_address), a(Y_address), 1)

    def upool2D_max(self, deltaX_address, X_address, IH, IW, deltaY_address, Y_address, OH, OW, FH, FW, N, IC, sh, sw, ph, pw):
        a = self._addr
        self._pool(self._lib.alpha_upool2D_max, N, IH, IW, IC, FH, FW, OH, OW, sh, sw, ph, pw, a(deltaY_address), a(Y_address),
                   a(X_address), a(deltaX_address))

    def upool2D_max_Indexed(self, deltaX_address, IH, IW, deltaY_address, Index_address, OH, OW, FH, FW, N, IC, sh, sw, ph, pw):
        a = self._addr
        self._pool(self._lib.alpha_upool2D_max_indexed, N, IH, IW, IC, FH, FW, OH, OW, sh, sw, ph, pw, a(deltaY_address),
                   a(Index_address), a(deltaX_address))

    def upool2D_avg(self, deltaX_address, IH, IW, deltaY_address, OH, OW, FH, FW, N, IC, sh, sw, ph, pw):
        a = self._addr
        self._pool(self._lib.alpha_upool2D_avg, N, IH, IW, IC, FH, FW, OH, OW, sh, sw, ph, pw, a(deltaY_address), a(deltaX_address), 0)

    def upool2D_avg_ignore_padding(self, deltaX_address, IH, IW, deltaY_address, OH, OW, FH, FW, N, IC, sh, sw, ph, pw):
        a = self._addr
        self._pool(self._lib.alpha_upool2D_avg, N, IH, IW, IC, FH, FW, OH, OW, sh, sw, ph, pw, a(deltaY_address), a(deltaX_address), 1)


def _pad4(n):
    return (n + 3) & ~3


def _pad_last(t, c4):
    """Copy of t whose last dimension is zero-padded to c4 (Tensor.java:208-221 memory rule)."""
    if t.dim() == 1:
        return _pad_both(t.reshape(1, -1), 1, c4).reshape(-1)
    return _pad_both(t, t.shape[0], c4)


def _pad_both(t, n4, c4):
    """t with its first dimension zero-padded to n4 and its last to c4 (contiguous; t itself where nothing is to pad)."""
    t = t.contiguous()
    shape = tuple(t.shape)
    if shape[-1] == c4 and shape[0] == n4:
        return t
    if t.dtype != torch.float32 or not t.is_cuda or t.numel() == 0 or t.is_neg():   # (a lazily negated view: its memory is not its value)
        out = torch.zeros((n4,) + shape[1:-1] + (c4,), dtype=t.dtype, device=t.device)
        out[: shape[0], ..., : shape[-1]] = t
        return out
    out = t.new_empty((n4,) + shape[1:-1] + (c4,))
    rows = t.numel() // shape[-1]
    with torch.cuda.device(t.device) if t.device.index != torch.cuda.current_device() else contextlib.nullcontext():
        _l.check(_l.load().alpha_pad_rows(t.data_ptr(), rows, shape[-1], out.data_ptr(), rows // shape[0] * n4, c4, _stream()))
    return out




@functools.lru_cache(maxsize=64)
def _adamw_rows(n):
    """n AlphaAdamW rows."""
    return struct.Struct("@" + "7Pqd4i" * n)


_dtype_of, _shape_of = operator.attrgetter("dtype"), operator.attrgetter("shape")
_FC_TYPES = {torch.float32: _l.ALPHA_F32, torch.bfloat16: _l.ALPHA_BF16, torch.float16: _l.ALPHA_F16}


def _fc_pack(dtype, *jobs):
    """The operands of one call, (t, groups, rows, cols, rows4, cols4) each: t holds `groups` matrices of rows x cols, wanted dense, on a 16-byte
    boundary and zero-padded to rows4 x cols4.  Those that need padding are written by one launch into one block of memory.  Returns addresses (None for
    None) and what has to be held until the call has been enqueued."""
    out, held, plan, size = [], [], [], 0
    for t, groups, rows, cols, rows4, cols4 in jobs:
        if t is None:
            out.append(None)
            continue
        if not t.is_contiguous():
            t = t.contiguous()
            held.append(t)
        if t.is_neg():                      # (a lazily negated view: its memory is not its value)
            t = t.resolve_neg()
            held.append(t)
        at = t.data_ptr()
        if cols != cols4 or rows != rows4:
            plan.append((len(out), at, groups, rows, cols, rows4, cols4, size, t))
            size += (groups * rows4 * cols4 + 127) // 128 * 128     # (each starts on 256 bytes, like a tensor of its own)
        elif at & 15:
            t = t.clone()
            held.append(t)
            at = t.data_ptr()
        out.append(at)
    if plan:
        block = torch.empty(size, dtype=dtype, device=plan[0][8].device)
        base, each, values = block.data_ptr(), block.element_size(), []
        for i, src, groups, rows, cols, rows4, cols4, at, _ in plan:
            out[i] = to = base + at * each
            for _ in range(groups):
                values += (src, rows, cols, to, rows4, cols4)
                src += rows * cols * each
                to += rows4 * cols4 * each
        _l.check(_l.load().alpha_pad_rows_typed(len(values) // 6, struct.pack("%dq" % len(values), *values), _FC_TYPES[dtype], _stream()))
        held.append(block)
    return out, held


@functools.lru_cache(maxsize=512)
def _fc_plan(what, glu, xs, ws, dtype):
    """Sizes of a FullConnect call on X of shape xs and W of shape ws: IC, OC, padded IC and OC, rows, halves of W, shapes of Y, Z and a
    bias."""
    if dtype not in _FC_TYPES:
        raise ValueError("%s: float32, bfloat16 or float16 tensors, not %s" % (what, dtype))
    if len(xs) < 1 or len(ws) != 2 or ws[1] != xs[-1]:
        raise ValueError("%s: X %s against W %s" % (what, tuple(xs), tuple(ws)))
    if glu and ws[0] % 2:
        raise ValueError("%s: W has %d rows, which are not gate rows and as many up rows" % (what, ws[0]))
    IC, halves = xs[-1], 2 if glu else 1
    OC, lead = ws[0] // halves, tuple(xs[:-1])
    if IC == 0 or OC == 0:
        raise ValueError("%s: X %s against W %s" % (what, tuple(xs), tuple(ws)))
    rows, unit = 1, 4 if dtype == torch.float32 else 8
    for n in lead:
        rows *= n
    if max(rows, IC, OC) > 2 ** 31 - 1024:       # (an int of the library's)
        raise ValueError("%s: X %s against W %s is too large" % (what, tuple(xs), tuple(ws)))
    return IC, OC, -(-IC // unit) * unit, -(-OC // 8) * 8, rows, halves, lead + (OC,), lead + (halves * OC,), (halves * OC,)


def _fc_check(what, X, W, others):
    """The tensors of a call are of X's type and on its GPU, and of the shapes expected: (name, tensor or None, shape) each.  Returns the GPU."""
    dtype, device = X.dtype, X.get_device()
    if device < 0:
        raise ValueError("%s: tensors must be on a GPU" % what)
    if W.dtype != dtype or W.get_device() != device:
        others += (("W", W, W.shape),)
    for name, t, shape in others:
        if t is None:
            continue
        if t.shape != shape:
            raise ValueError("%s: %s %s, expected %s" % (what, name, tuple(t.shape), shape))
        if t.dtype != dtype or t.get_device() != device:
            raise ValueError("%s: %s is %s on %s, X %s on %s" % (what, name, t.dtype, t.device, dtype, X.device))
    return device


def _fc_act(what, act):
    code = _l.ACTS.get(act)
    if code is None:
        raise ValueError("%s: act must be one of %s, not %r" % (what, ", ".join(sorted(_l.ACTS)), act))
    return code


def _same_memory(g, o):
    return g is o or (g.data_ptr() == o.data_ptr() and g.dtype == o.dtype and g.shape == o.shape and g.stride() == o.stride() and g.is_neg() == o.is_neg())


def _memory_of(t):
    """Where a tensor lies: its first byte, the byte after its last, and, if its elements are rows of `wide` bytes `pitch` apart, these (else 0, 0; a dense tensor
    is one row).  None where elements may share memory."""
    dims = sorted((st, n) for n, st in zip(t.shape, t.stride()) if n > 1)
    size, wide, pitch, reach = t.element_size(), 1, 0, 1         # in elements; reach: from the first to after the last
    for st, n in dims:
        if st < reach:
            return None
        if not pitch and st == wide:
            wide *= n
        elif not pitch:
            pitch, rows = st, n
        elif st == pitch * rows:
            rows *= n
        else:
            pitch = -1
        reach += (n - 1) * st
    at = t.data_ptr()
    if pitch < 0:
        return at, at + reach * size, 0, 0
    return at, at + reach * size, wide * size, pitch * size


def _apart(a, b):
    """Whether two tensors (_memory_of) share no byte, as far as can be told: disjoint, or columns of rows of one pitch."""
    if a[0] > b[0]:
        a, b = b, a
    if a[1] <= b[0]:
        return True
    if not a[2] or not b[2] or (a[3] and b[3] and a[3] != b[3]):
        return False
    pitch, d = a[3] or b[3], b[0] - a[0]
    if not pitch or (not a[3] and a[2] > pitch) or (not b[3] and b[2] > pitch):
        return False
    d %= pitch
    return d >= a[2] and d + b[2] <= pitch


def _refuse_overlaps(what, grads, Out):
    """Raises where an output overlaps itself, another output or a gradient that is not its own (as the library does for dense tensors)."""
    places = []                          # (place, written)
    for g, o in zip(grads, Out):
        if o.numel() == 0:
            continue
        place = _memory_of(o)
        if place is None:
            raise ValueError("%s: elements of an output share memory" % what)
        places.append((place, True))
        if not _same_memory(g, o):
            places.append((_memory_of(g) or (g.data_ptr(), g.data_ptr() + g.element_size() * (1 + sum((n - 1) * st for n, st in zip(g.shape, g.stride()))), 0, 0), False))
    places.sort()
    for i, (a, write) in enumerate(places):
        for b, other in itertools.islice(places, i + 1, None):
            if b[0] >= a[1]:
                break
            if (write or other) and not _apart(a, b):
                raise ValueError("%s: an output overlaps another tensor" % what)


def _dense(t):
    """t as dense memory that holds its values."""
    return t.resolve_neg().contiguous()


def _present(tensors):
    """Those of a list that are not None: the list itself where all are."""
    return [t for t in tensors if t is not None] if type(None) in set(map(type, tensors)) else tensors


def _dense_now(t):
    """The same without a call where there is nothing to do (None: None)."""
    return t if t is None or (t.is_contiguous() and not t.is_neg()) else _dense(t.detach())


@functools.lru_cache(maxsize=512)
def _norm_plan(what, shape, groups, dtype, affine, act, k, eps):
    """The library's shape of a group normalisation and that of its means, or None where X holds no samples."""
    if dtype not in _FC_TYPES:
        raise ValueError("%s: float32, bfloat16 or float16 tensors, not %s" % (what, dtype))
    if len(shape) < 2 or groups < 1 or shape[-1] < 1 or shape[-1] % groups:
        raise ValueError("%s: X %s in %d groups of channels" % (what, tuple(shape), groups))
    if affine not in (None, dtype, torch.float32):
        raise ValueError("%s: gamma and beta are %s, X %s" % (what, affine, dtype))
    positions = 1
    for n in shape[1:-1]:
        positions *= n
    if positions == 0:
        raise ValueError("%s: X %s has no positions to take a mean of" % (what, tuple(shape)))
    if shape[0] == 0:
        return None
    if max(shape[0] * shape[-1], positions) >= 2 ** 31:
        raise ValueError("%s: X %s is too large" % (what, tuple(shape)))
    return _l.AlphaNormShape(shape[0], positions, shape[-1], groups, _FC_TYPES[dtype], _FC_TYPES[affine or dtype], act, k, eps), (shape[0], groups)


class AdamWState:
    """The moments of Engine.adamW, a list of each: float32 tensors of the parameters' shapes, or (8 bits) float8_e4m3fn codes of these shapes with
    float8_e8m0fnu scales, one for every 32 elements in the order they lie in.  Engine.adamW_state makes one; a program that keeps its moments elsewhere (views of a flat
    buffer, a checkpoint) passes its own dense tensors."""

    def __init__(self, m, v, m_scale=None, v_scale=None):
        self.m, self.v = list(m), list(v)
        if (m_scale is None) != (v_scale is None):
            raise ValueError("AdamWState: scales of both moments, or of neither")
        self.m_scale, self.v_scale = (None, None) if m_scale is None else (list(m_scale), list(v_scale))
        self.bits = 32 if m_scale is None else 8
        lists = [self.m, self.v] + ([self.m_scale, self.v_scale] if self.bits == 8 else [])
        if len(set(map(len, lists))) != 1:
            raise ValueError("AdamWState: lists of different lengths")
        code = torch.float32 if self.bits == 32 else torch.float8_e4m3fn
        for i, (a, b) in enumerate(zip(self.m, self.v)):
            if a.dtype != code or b.dtype != code or a.shape != b.shape:
                raise ValueError("AdamWState: moments of tensor %d are %s %s and %s %s, expected %s of one shape" % (i, a.dtype, tuple(a.shape), b.dtype, tuple(b.shape), code))
        if self.bits == 8:
            for i, (a, s, t) in enumerate(zip(self.m, self.m_scale, self.v_scale)):
                if any(x.dtype != torch.float8_e8m0fnu or x.numel() != -(-a.numel() // 32) for x in (s, t)):
                    raise ValueError("AdamWState: scales of tensor %d must be %d float8_e8m0fnu values" % (i, -(-a.numel() // 32)))
        for t in itertools.chain.from_iterable(lists):
            if not t.is_contiguous() or t.is_neg():
                raise ValueError("AdamWState: moments must be dense")


_pack_jobs = {n: struct.Struct("%dq" % (6 * n)).pack for n in (1, 2, 3)}


def _pad_all(*jobs):
    """_pad_both for the tensors of one call, (t, n4, c4) each: those that need padding are written by one launch into one block of memory.
    Returns tensors, or addresses inside the block, and the block (to be held until the call has been enqueued)."""
    for t, n4, c4 in jobs:
        shape = t.shape
        if shape[-1] != c4 or shape[0] != n4:
            break
    else:
        return [job[0].contiguous() for job in jobs], None
    out = [job[0] for job in jobs]
    odd = [i for i, (t, n4, c4) in enumerate(jobs) if t.shape[-1] != c4 or t.shape[0] != n4]
    device = out[odd[0]].device
    if device.type != "cuda" or device.index != torch.cuda.current_device() or any(
            out[i].dtype != torch.float32 or out[i].device != device or out[i].numel() == 0 or out[i].is_neg() for i in odd):
        return [_pad_both(*job) for job in jobs], None
    plan, size = [], 0
    for i in odd:
        t, n4, c4 = jobs[i]
        t = t.contiguous()
        n, c = t.shape[0], t.shape[-1]
        rows = t.numel() // c
        plan.append((i, t, rows, c, size, rows // n * n4, c4))
        size += (rows // n * n4 * c4 + 63) // 64 * 64          # (each starts on 256 bytes, like a tensor of its own)
    block = out[odd[0]].new_empty(size)
    base = block.data_ptr()
    _l.check(_l.load().alpha_pad_rows_many(len(plan), _pack_jobs[len(plan)](
        *[v for _, t, rows, c, at, rows4, c4 in plan for v in (t.data_ptr(), rows, c, base + 4 * at, rows4, c4)]), _stream()))
    for i, _, _, _, at, _, _ in plan:
        out[i] = base + 4 * at
    return [t.contiguous() if isinstance(t, torch.Tensor) else t for t in out], block


class Engine:
    """Tensor-level conv operators (Engine.java:1541, 1601, 1697, 1788) on torch CUDA tensors.

    Tensors are NHWC float32.  Channel counts and the batch that are not multiples of 4 are padded
    with zero lanes exactly as Dragon-Alpha's Tensor memory layout does, and sliced back.
    """

    def __init__(self, base=None):
        self.base = base if base is not None else CudaFloat32EngineBase()

    @staticmethod
    def out_size(IH, IW, FH, FW, sh, sw, ph, pw):
        return (IH - FH + 2 * ph) // sh + 1, (IW - FW + 2 * pw) // sw + 1

    def conv3D(self, X, W, sh, sw, ph, pw, Bias=None):
        N, IH, IW, IC = X.shape
        OC, FH, FW, WIC = W.shape
        if WIC != IC:
            raise ValueError("W.IC=%d != X.IC=%d" % (WIC, IC))
        OH, OW = self.out_size(IH, IW, FH, FW, sh, sw, ph, pw)
        ic4, oc4 = _pad4(IC), _pad4(OC)
        Y = _new(X, (N, OH, OW, oc4))
        if Bias is None:
            (Xp, Wp), _held = _pad_all((X, N, ic4), (W, oc4, ic4))
            self.base.conv3D(Y, OH, OW, Xp, IH, IW, Wp, FH, FW, N, ic4, oc4, sh, sw, ph, pw)
        else:
            (Xp, Wp, Bp), _held = _pad_all((X, N, ic4), (W, oc4, ic4), (Bias.reshape(1, -1), 1, oc4))
            self.base.conv3D_biased(Y, OH, OW, Xp, IH, IW, Wp, FH, FW, Bp, N, ic4, oc4, sh, sw, ph, pw)
        return Y if oc4 == OC else Y[..., :OC]

    def conv3D_biased(self, X, W, Bias, sh, sw, ph, pw):
        return self.conv3D(X, W, sh, sw, ph, pw, Bias=Bias)

    def conv3D_leakyRelu(self, X, W, Bias, k, sh, sw, ph, pw):
        """leakyRelu(conv3D(_biased)(X, W[, Bias]), k) with the activation in the kernel's epilogue: what a
        Conv3D unit followed by a LeakyRelu unit computes (Engine.leakyRelu, Cuda_function's
        leakyRelu2D); k = 0 is relu."""
        N, IH, IW, IC = X.shape
        OC, FH, FW, WIC = W.shape
        if WIC != IC:
            raise ValueError("W.IC=%d != X.IC=%d" % (WIC, IC))
        OH, OW = self.out_size(IH, IW, FH, FW, sh, sw, ph, pw)
        ic4, oc4 = _pad4(IC), _pad4(OC)
        bias = () if Bias is None else ((Bias.reshape(1, -1), 1, oc4),)
        (Xp, Wp, *Bp), _held = _pad_all((X, N, ic4), (W, oc4, ic4), *bias)
        Bp = Bp[0] if Bp else None
        Y = _new(X, (N, OH, OW, oc4))
        shape = _conv_shape(N, IH, IW, ic4, oc4, FH, FW, OH, OW, sh, sw, ph, pw)
        a = self.base._addr
        _l.check(self.base._lib.alpha_conv3d_forward_leakyRelu(C.byref(shape), a(Xp), a(Wp), a(Bp) if Bp is not None else None,
                                                               float(k), a(Y), _stream(self.base._stream)))
        return Y if oc4 == OC else Y[..., :OC]

    def field_sum(self, X, row_length=-1):
        """Engine.field_sum(X, row_length) (Engine.java:6945): sums the rows of X seen as a matrix of
        `row_length` columns; Conv3D.__backward__ calls it on deltaY with OC for the bias gradient."""
        if row_length == -1:
            row_length = X.shape[-1]
        if X.shape[-1] != row_length:
            raise ValueError("field_sum: row_length must be the last dimension")
        oc4 = _pad4(row_length)
        Xp = _pad_last(X, oc4).contiguous()
        out = _new(X, (oc4,))
        rows = Xp.numel() // oc4
        _l.check(self.base._lib.alpha_conv_bias_grad(self.base._addr(Xp), rows, oc4, self.base._addr(out),
                                                     _stream(self.base._stream)))
        return out if oc4 == row_length else out[:row_length]

    def dconv3D_deltaW(self, X, deltaY, FH, FW, sh, sw, ph, pw):
        N, IH, IW, IC = X.shape
        _, OH, OW, OC = deltaY.shape
        ic4, oc4 = _pad4(IC), _pad4(OC)
        (Xp, dYp), _held = _pad_all((X, N, ic4), (deltaY, deltaY.shape[0], oc4))
        dW = _new(X, (oc4, FH, FW, ic4))
        self.base.dconv3D_deltaW(dW, FH, FW, Xp, IH, IW, dYp, OH, OW, N, ic4, oc4, sh, sw, ph, pw)
        return dW if (ic4 == IC and oc4 == OC) else dW[:OC, :, :, :IC]

    def dconv3D_deltaW_bias(self, X, deltaY, FH, FW, sh, sw, ph, pw):
        """(deltaW, deltaB) of a biased Conv3D unit in one call: dconv3D_deltaW and field_sum(deltaY, OC) of
        Conv3D.__backward__ (nn/unit/simple/Conv3D.java:150-160); stride-1 layers sum the bias columns inside
        the deltaW kernel's pass over deltaY."""
        N, IH, IW, IC = X.shape
        _, OH, OW, OC = deltaY.shape
        ic4, oc4 = _pad4(IC), _pad4(OC)
        (Xp, dYp), _held = _pad_all((X, N, ic4), (deltaY, deltaY.shape[0], oc4))
        dW = _new(X, (oc4, FH, FW, ic4))
        dB = _new(X, (oc4,))
        shape = _conv_shape(N, IH, IW, ic4, oc4, FH, FW, OH, OW, sh, sw, ph, pw)
        a = self.base._addr
        _l.check(self.base._lib.alpha_conv3d_deltaW_bias(C.byref(shape), a(Xp), a(dYp), a(dW), a(dB), _stream(self.base._stream)))
        return (dW if (ic4 == IC and oc4 == OC) else dW[:OC, :, :, :IC]), (dB if oc4 == OC else dB[:OC])

    def dconv3D_deltaX(self, deltaY, W, IH, IW, sh, sw, ph, pw):
        N, OH, OW, OC = deltaY.shape
        _, FH, FW, IC = W.shape
        ic4, oc4 = _pad4(IC), _pad4(OC)
        (dYp, Wp), _held = _pad_all((deltaY, N, oc4), (W, oc4, ic4))
        dX = _new(deltaY, (N, IH, IW, ic4))
        self.base.dconv3D_deltaX(dX, IH, IW, dYp, OH, OW, Wp, FH, FW, N, ic4, oc4, sh, sw, ph, pw)
        return dX if ic4 == IC else dX[..., :IC]

    # ---- matrix products (Engine.matMul / matMulT1 / matMulT2, Engine.java) -------------------------------
    def matMul(self, A, B, Bias=None):
        """C[N,M] = A[N,K] * B[K,M] (+ Bias[M] per row); dimensions are zero-padded to multiples of 4 as the
        engine's tensor memory is, and sliced back."""
        (N, K), (K2, M) = A.shape, B.shape
        if K != K2:
            raise ValueError("A.width=%d != B.height=%d" % (K, K2))
        n4, k4, m4 = _pad4(N), _pad4(K), _pad4(M)
        C = _new(A, (n4, m4))
        if Bias is None:
            (Ap, Bp), _held = _pad_all((A, n4, k4), (B, k4, m4))
            self.base.matMul(C, Ap, Bp, n4, m4, k4)
        else:
            (Ap, Bp, bp), _held = _pad_all((A, n4, k4), (B, k4, m4), (Bias.reshape(1, -1), 1, m4))
            self.base.matMul_biased(C, Ap, Bp, n4, m4, k4, bp)
        return C[:N, :M]

    def matMulT1(self, A, B):
        """C[N,M] = A[K,N]^T * B[K,M]."""
        (K, N), (K2, M) = A.shape, B.shape
        if K != K2:
            raise ValueError("A.height=%d != B.height=%d" % (K, K2))
        n4, k4, m4 = _pad4(N), _pad4(K), _pad4(M)
        (Ap, Bp), _held = _pad_all((A, k4, n4), (B, k4, m4))
        C = _new(A, (n4, m4))
        self.base.matMulT1(C, Ap, Bp, n4, m4, k4)
        return C[:N, :M]

    def matMulT2(self, A, B):
        """C[N,M] = A[N,K] * B[M,K]^T."""
        (N, K), (M, K2) = A.shape, B.shape
        if K != K2:
            raise ValueError("A.width=%d != B.width=%d" % (K, K2))
        n4, k4, m4 = _pad4(N), _pad4(K), _pad4(M)
        (Ap, Bp), _held = _pad_all((A, n4, k4), (B, m4, k4))
        C = _new(A, (n4, m4))
        self.base.matMulT2(C, Ap, Bp, n4, m4, k4)
        return C[:N, :M]

    # ---- FullConnect layers of a transformer: the product with bias, activation and residual in its epilogue, the gated block, their
    # gradients.  float32, bfloat16 or float16 tensors (all of one type); X may have any leading dimensions; IC that is no multiple of 16 bytes
    # is zero-padded as everywhere, and so are tensors of OC columns that is no multiple of 8 (not W). ----
    def _fc_forward(self, what, X, W, Bias, act, k, Residual, save, glu):
        plan = _fc_plan(what, glu, X.shape, W.shape, X.dtype)
        code = _fc_act(what, act)
        device = _fc_check(what, X, W, (("Bias", Bias, plan[8]), ("Residual", Residual, plan[6])) if Bias is not None or Residual is not None else ())
        if self.base._stream is None and device == torch._C._cuda_getDevice():
            return self._fc_run(X, W, Bias, code, k, Residual, save, glu, plan)
        with self._on(X):
            return self._fc_run(X, W, Bias, code, k, Residual, save, glu, plan)

    def _fc_run(self, X, W, Bias, code, k, Residual, save, glu, plan):
        IC, OC, ic, oc, rows, halves, ys, zs, _ = plan
        dtype = X.dtype
        if rows == 0:
            return (X.new_empty(ys), X.new_empty(zs)) if save else X.new_empty(ys)
        (Xp, Wp, Bp, Rp), _held = _fc_pack(dtype, (X, 1, rows, IC, rows, ic), (W, 1, halves * OC, IC, halves * OC, ic), (Bias, 1, halves, OC, halves, oc), (Residual, 1, rows, OC, rows, oc))
        even = oc == OC
        Y = X.new_empty(ys if even else (rows, oc))
        Z = X.new_empty(zs if even else (rows, halves * oc)) if save else None
        if glu:
            self.base.fullConnect_glu(Y.data_ptr(), Xp, Wp, rows, ic, OC, _FC_TYPES[dtype], code, k, Bp, Z)
        else:
            self.base.fullConnect(Y.data_ptr(), Xp, Wp, rows, ic, OC, _FC_TYPES[dtype], code, k, Bp, Rp, Z)
        if not even:
            Y = Y.narrow(1, 0, OC)
            if len(ys) != 2:
                Y = Y.reshape(ys)
            if save:
                Z = Z.reshape(rows, 2, oc)[:, :, :OC].reshape(zs) if glu else Z.narrow(1, 0, OC).reshape(zs)
        return (Y, Z) if save else Y

    def _fc_delta(self, what, deltaY, X, W, Z, act, k, bias, glu):
        plan = _fc_plan(what, glu, X.shape, W.shape, X.dtype)
        code = _fc_act(what, act)
        device = _fc_check(what, X, W, (("deltaY", deltaY, plan[6]), ("Z", Z, plan[7])))
        if Z is None and (glu or act != "none"):
            raise ValueError("%s: Z of the forward pass is needed" % what)
        if self.base._stream is None and device == torch._C._cuda_getDevice():
            return self._fc_run_delta(deltaY, X, W, Z, code, k, bias, glu, plan)
        with self._on(X):
            return self._fc_run_delta(deltaY, X, W, Z, code, k, bias, glu, plan)

    def _fc_run_delta(self, deltaY, X, W, Z, code, k, bias, glu, plan):
        IC, OC, ic, oc, rows, halves, _, _, _ = plan
        dtype = X.dtype
        if rows == 0:
            return X.new_empty(X.shape), W.new_zeros(W.shape), W.new_zeros((halves * OC,)) if bias else None
        through = glu or code != 0
        (dYp, Xp, Wp, Zp), _held = _fc_pack(dtype, (deltaY, 1, rows, OC, rows, oc), (X, 1, rows, IC, rows, ic), (W, 1, halves * OC, IC, halves * OC, ic),
                                            (Z if through else None, 1, rows * halves, OC, rows * halves, oc))
        dZ = X.new_empty((rows, halves * oc)) if through else None
        dX, dW = X.new_empty((rows, ic)), W.new_empty((halves * OC, ic))
        dB = W.new_empty((halves, oc)) if bias else None
        self.base.fullConnect_delta(dX, dW, dB, dYp, Xp, Wp, Zp, dZ, rows, ic, OC, _FC_TYPES[dtype], code, k, glu)
        if ic != IC:
            dX, dW = dX.narrow(1, 0, IC), dW.narrow(1, 0, IC)
        if bias:
            dB = (dB if oc == OC else dB.narrow(1, 0, OC)).reshape(halves * OC)
        return dX if X.dim() == 2 else dX.reshape(X.shape), dW, dB

    def fullConnect(self, X, W, Bias=None, act="none", k=0.0, Residual=None, save=False):
        """act(X W^T + Bias) + Residual in one pass; W [OC, IC], X [..., IC].  act: 'none', 'leakyRelu' (slope k; relu k = 0),
        'sigmoid', 'silu', 'gelu' (of the normal distribution function) or 'gelu_tanh'.  save=True also returns
        Z = X W^T + Bias, which fullConnect_delta reads."""
        return self._fc_forward("fullConnect", X, W, Bias, act, k, Residual, save, False)

    def fullConnect_delta(self, deltaY, X, W, Z=None, act="none", k=0.0, bias=False):
        """(deltaX, deltaW, deltaB) of fullConnect from deltaY and its Z (not needed with act 'none'); deltaB is None without
        bias=True.  The gradient of a residual is deltaY itself."""
        return self._fc_delta("fullConnect_delta", deltaY, X, W, Z, act, k, bias, False)

    def fullConnect_glu(self, X, W, Bias=None, act="silu", k=0.0, save=False):
        """The gated block act(G) * U with [G | U] = Z = X W^T + Bias in one pass; W [2 OC, IC]: the gate rows, then the up rows.
        save=True also returns Z, which fullConnect_glu_delta reads."""
        return self._fc_forward("fullConnect_glu", X, W, Bias, act, k, None, save, True)

    def fullConnect_glu_delta(self, deltaY, X, W, Z, act="silu", k=0.0, bias=False):
        """(deltaX, deltaW, deltaB) of fullConnect_glu from deltaY and its Z; deltaB is None without bias=True."""
        return self._fc_delta("fullConnect_glu_delta", deltaY, X, W, Z, act, k, bias, True)

    # ---- the loss on top of such a layer ----
    def _loss_call(self, what, X, W, label, Bias, others):
        """The checked call's plan."""
        plan = _fc_plan(what, False, X.shape, W.shape, X.dtype)
        device = _fc_check(what, X, W, (("Bias", Bias, plan[8]),) if Bias is not None else ())
        lead = X.shape[:-1]
        if label.dtype not in (torch.int64, torch.int32):
            raise ValueError("%s: label must be int64 or int32, not %s" % (what, label.dtype))
        for name, t in (("label", label),) + others:
            if t.shape != lead or t.get_device() != device:
                raise ValueError("%s: %s %s on %s, expected %s on %s" % (what, name, tuple(t.shape), t.device, tuple(lead), X.device))
            if name != "label" and t.dtype != torch.float32:
                raise ValueError("%s: %s must be float32, not %s" % (what, name, t.dtype))
        return plan

    def fullConnect_softmax_crossEntropy(self, X, W, label, Bias=None, save=False):
        """The softmax cross entropy of every row of X [..., IC] over the classes of a FullConnect layer, logsumexp(z) - z[label] with z = X W^T + Bias, as float32 [...].
        The logits are not kept.  W [OC, IC]; label [...] int64 or int32; a row whose label is not in [0, OC) does not count: its loss is 0.  save=True also returns
        the logsumexp of every row, which fullConnect_softmax_crossEntropy_delta reads."""
        plan = self._loss_call("fullConnect_softmax_crossEntropy", X, W, label, Bias, ())
        if self.base._stream is None and X.get_device() == torch._C._cuda_getDevice():
            return self._loss_run(plan, X, W, label, Bias, save)
        with self._on(X):
            return self._loss_run(plan, X, W, label, Bias, save)

    def _loss_run(self, plan, X, W, label, Bias, save):
        IC, OC, ic, oc, rows = plan[:5]
        dtype, lead = X.dtype, X.shape[:-1]
        loss = _new(X, lead)
        lse = _new(X, lead) if save else None
        if rows:
            (Xp, Wp, Bp), _held = _fc_pack(dtype, (X, 1, rows, IC, rows, ic), (W, 1, OC, IC, OC, ic), (Bias, 1, 1, OC, 1, oc))
            label = _dense_now(label)
            self.base.fullConnect_softmax_crossEntropy(loss.data_ptr(), lse, Xp, Wp, Bp, label.data_ptr(), label.element_size(), rows, ic, OC, _FC_TYPES[dtype])
        return (loss, lse) if save else loss

    def fullConnect_softmax_crossEntropy_delta(self, deltaL, X, W, label, lse, Bias=None):
        """(deltaX, deltaW, deltaB) of fullConnect_softmax_crossEntropy from the gradients of the rows' losses and the lse it saved; deltaB is None without Bias.  deltaL: float32 of
        the losses' shape, or one number for all (a float, or a tensor of one float32 value)."""
        what = "fullConnect_softmax_crossEntropy_delta"
        step = 0
        if isinstance(deltaL, torch.Tensor) and (deltaL.dim() or X.dim() == 1):
            step = 1
        plan = self._loss_call(what, X, W, label, Bias, (("lse", lse),) + ((("deltaL", deltaL),) if step else ()))
        if not step and isinstance(deltaL, torch.Tensor) and (deltaL.dtype != torch.float32 or deltaL.get_device() != X.get_device()):
            raise ValueError("%s: deltaL must be float32 on %s, not %s on %s" % (what, X.device, deltaL.dtype, deltaL.device))
        if self.base._stream is None and X.get_device() == torch._C._cuda_getDevice():
            return self._loss_run_delta(plan, deltaL, step, X, W, label, lse, Bias)
        with self._on(X):
            return self._loss_run_delta(plan, deltaL, step, X, W, label, lse, Bias)

    def _loss_run_delta(self, plan, deltaL, step, X, W, label, lse, Bias):
        IC, OC, ic, oc, rows = plan[:5]
        dtype = X.dtype
        if rows == 0:
            return X.new_empty(X.shape), W.new_zeros(W.shape), None if Bias is None else W.new_zeros((OC,))
        if not isinstance(deltaL, torch.Tensor):
            deltaL = X.new_full((), float(deltaL), dtype=torch.float32)
        (Xp, Wp, Bp), _held = _fc_pack(dtype, (X, 1, rows, IC, rows, ic), (W, 1, OC, IC, OC, ic), (Bias, 1, 1, OC, 1, oc))
        label, lse, deltaL = _dense_now(label), _dense_now(lse), _dense_now(deltaL)
        dX, dW = X.new_empty((rows, ic)), W.new_empty((OC, ic))
        dB = None if Bias is None else W.new_empty((oc,))
        self.base.fullConnect_softmax_crossEntropy_delta(dX.data_ptr(), dW.data_ptr(), dB, deltaL.data_ptr(), step, Xp, Wp, Bp, label.data_ptr(), label.element_size(), lse.data_ptr(),
                                                         rows, ic, OC, _FC_TYPES[dtype])
        if ic != IC:
            dX, dW = dX.narrow(1, 0, IC), dW.narrow(1, 0, IC)
        return dX if X.dim() == 2 else dX.reshape(X.shape), dW, None if dB is None else dB if oc == OC else dB.narrow(0, 0, OC)

    # ---- all gradients of a step ----
    def _on(self, t):
        """t's device as the current one and, where the engine has a stream of its own, that as the current one: copies and memory of
        the call then belong to the stream its kernels run on."""
        s = self.base._stream
        if s is not None:
            if s.device != t.device:
                raise ValueError("the engine's stream is on %s, the tensors on %s" % (s.device, t.device))
            return torch.cuda.stream(s)
        return torch.cuda.device(t.device) if t.device.index != torch.cuda.current_device() else contextlib.nullcontext()

    @staticmethod
    def _check_grads(what, grads, Out):
        """Raises for tensors the library would not read, else returns (all of them, their type codes, whether all are dense)."""
        # (a pass over all tensors for each question: half the time of a loop that asks them one by one)
        T, device, both = torch.Tensor, grads[0].get_device(), grads if Out is grads else grads + Out
        codes = list(map(_FC_TYPES.get, map(_dtype_of, both)))
        if (device < 0 or set(map(T.get_device, both)) != {device} or None in codes
                or (both is not grads and list(map(_shape_of, grads)) != list(map(_shape_of, Out)))):
            for g, o in zip(grads, Out):
                Engine._refuse_grads(what, device, g, o)
        return both, codes, all(map(T.is_contiguous, both)) and not any(map(T.is_neg, both))

    @staticmethod
    def _refuse_grads(what, device, g, o):
        """Raises for what is wrong with this pair, if anything."""
        if device < 0 or g.get_device() != device or o.get_device() != device:
            raise ValueError("%s: tensors must be on one GPU" % what)
        for t in (g, o):
            if t.dtype not in _FC_TYPES:
                raise ValueError("%s: float32, bfloat16 or float16 tensors, not %s" % (what, t.dtype))
        if g.shape != o.shape:
            raise ValueError("%s: gradient %s, output %s" % (what, tuple(g.shape), tuple(o.shape)))

    @staticmethod
    def _grad_table(n, both, codes):
        """The tensors as the table the library reads (AlphaGrad: two addresses, a count, two types)."""
        at = list(map(torch.Tensor.data_ptr, both))
        types = [g | o << 32 for g, o in zip(codes, codes[-n:])]
        return struct.pack("<%dq" % (4 * n), *itertools.chain.from_iterable(zip(at, at[-n:], map(torch.Tensor.numel, both), types)))

    @staticmethod
    def _dense_grads(what, grads, Out):
        """Dense copies of the tensors that are not (an output that is one gets its own), and the pairs (output, copy) to be copied back.  Such are the views that
        fullConnect_delta returns where IC is no multiple of 16 bytes."""
        _refuse_overlaps(what, grads, Out)
        dense, to, back = [], [], []
        for g, o in zip(grads, Out):
            same = _same_memory(g, o)
            d = g.resolve_neg().contiguous()
            if o.is_contiguous() and not o.is_neg():
                t = o
            elif same:
                t = d                                   # (a copy of its own: g is not dense)
            else:
                t = torch.empty(o.shape, dtype=o.dtype, device=o.device)
            if t is not o:
                back.append((o, t))
            dense.append(t if same else d)
            to.append(t)
        return dense, to, back

    def grad_norm(self, grads):
        """The 2-norm of all elements of a list of gradients (float32, bfloat16, float16) as a 0-dimensional float32 tensor."""
        grads = list(grads)
        if not grads:
            return torch.zeros((), device="cuda")
        both, codes, dense = self._check_grads("grad_norm", grads, grads)
        with self._on(grads[0]):
            if not dense:
                with torch.no_grad():
                    both = [g.resolve_neg().contiguous() for g in grads]
            norm = torch.empty((), dtype=torch.float32, device=grads[0].device)
            _l.check(self.base._lib.alpha_grad_norm(len(grads), self._grad_table(len(grads), both, codes), norm.data_ptr(), _stream(self.base._stream)))
        return norm

    def clip_grad_norm(self, grads, max_norm, Out=None):
        """grad_norm, and every gradient scaled by min(1, max_norm / (norm + 1e-6)): in place, or into the tensors of Out, which may
        be of another type.  Nothing waits for the norm on the host.  Tensors that are not dense go through copies; an output must not overlap itself or
        another tensor of the call."""
        grads = list(grads)
        Out = grads if Out is None else list(Out)
        if len(Out) != len(grads):
            raise ValueError("clip_grad_norm: %d gradients, %d outputs" % (len(grads), len(Out)))
        if not grads:
            return torch.zeros((), device="cuda")
        both, codes, dense = self._check_grads("clip_grad_norm", grads, Out)
        max_norm, back = float(max_norm), ()
        with self._on(grads[0]):
            if not dense:
                with torch.no_grad():
                    src, to, back = self._dense_grads("clip_grad_norm", grads, Out)
                both, codes = src + to, codes if len(codes) > len(grads) else codes + codes
            norm = torch.empty((), dtype=torch.float32, device=grads[0].device)
            _l.check(self.base._lib.alpha_clip_grad_norm(len(grads), self._grad_table(len(grads), both, codes), max_norm, norm.data_ptr(), _stream(self.base._stream)))
            if back:
                with torch.no_grad():
                    for o, t in back:
                        o.copy_(t)
        return norm

    # ---- the optimizer's step after them ----
    @staticmethod
    def adamW_state(params, bits=32):
        """Moments of 0 for the tensors of `params`, of 32 or 8 bits."""
        params = list(params)
        if bits == 32:
            return AdamWState(*([torch.zeros(p.shape, dtype=torch.float32, device=p.device) for p in params] for _ in range(2)))
        if bits != 8:
            raise ValueError("adamW_state: moments of 32 or 8 bits, not %r" % (bits,))
        codes, scales = ([[torch.zeros(shape(p), dtype=torch.uint8, device=p.device).view(t) for p in params] for _ in range(2)] for shape, t in (
            (lambda p: p.shape, torch.float8_e4m3fn), (lambda p: (-(-p.numel() // 32),), torch.float8_e8m0fnu)))
        return AdamWState(*codes, *scales)

    @staticmethod
    def _device_value(what, name, x, dtype, device):
        """(value, None) of a number, (0, address) of a tensor of one element on the GPU."""
        if not isinstance(x, torch.Tensor):
            return x, None
        if x.dtype != dtype or x.numel() != 1 or x.get_device() != device or x.is_neg():
            raise ValueError("%s: %s on the GPU must be one %s value beside the tensors" % (what, name, dtype))
        return 0, x.data_ptr()

    def adamW(self, params, grads, state, step, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, max_norm=None, norm=None, Out=None, seed=0):
        """One AdamW step in place over lists of parameters and gradients (float32, bfloat16, float16; those without a gradient, None, are left out)
        and their moments (AdamWState):  m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2,
            p = p (1 - lr weight_decay) - lr / (1 - beta1^step) m / (sqrt(v / (1 - beta2^step)) + eps).
        step (from 1 on) and lr may be tensors of one int64 and float32 value on the GPU, for a step that a graph replays; weight_decay one number or one for each tensor.
        max_norm: gradients are scaled by min(1, max_norm / (norm + 1e-6)) on the way, and not written; norm is that of grad_norm unless given (one float32 value on the
        GPU), and a step whose norm is NaN or Inf changes nothing.  Out: tensors of the parameters' shapes (None: none) that take the new values in their own type, the 16-bit
        copies of float32 weights.  seed (32 bits): of the rounding of 8-bit moments.  Returns the norm, or None without max_norm."""
        what, params, grads = "adamW", list(params), list(grads)
        n = len(params)
        outs = None if Out is None else list(Out)
        decay = [float(weight_decay)] * n if not isinstance(weight_decay, (list, tuple)) else list(map(float, weight_decay))
        if len(grads) != n or len(decay) != n or len(state.m) != n or (outs is not None and len(outs) != n):
            raise ValueError("adamW: %d parameters, %d gradients, moments of %d, %s outputs, %d weight decays" % (n, len(grads), len(state.m), n if outs is None else len(outs), len(decay)))
        if norm is not None and max_norm is None:
            raise ValueError("adamW: a norm without max_norm")
        seed = operator.index(seed)
        if not 0 <= seed < 2 ** 32:
            raise ValueError("adamW: seed must have 32 bits")
        used = _present(grads)
        if not used:
            return None if max_norm is None else norm if norm is not None else self.grad_norm([])
        eight = state.bits == 8
        lists = [state.m, state.v] + ([state.m_scale, state.v_scale] if eight else [])
        device, dense = self._check_adamw(what, params, grads, outs, lists)
        lr, lr_at = self._device_value(what, "lr", lr, torch.float32, device)
        step, step_at = self._device_value(what, "step", step, torch.int64, device)
        with self._on(used[0]), torch.no_grad():
            if not dense:
                grads = [None if g is None else _dense(g) for g in grads]
                used = _present(grads)
            norm_at = None
            if max_norm is not None:
                if norm is None:
                    norm = self.grad_norm(used)
                norm_at = self._device_value(what, "norm", norm, torch.float32, device)[1]
                if norm_at is None:
                    raise ValueError("adamW: norm must be a tensor on the GPU")
            # a tensor without a gradient has a row of no elements: the others keep their numbers, which the random bits of their moments go by
            at, code, none = torch.Tensor.data_ptr, _FC_TYPES.__getitem__, itertools.repeat(0)
            if len(used) == n:
                g_at, g_code, count = map(at, grads), map(code, map(_dtype_of, grads)), map(torch.Tensor.numel, params)
            else:
                g_at, g_code, count = ([0 if g is None else f(x) for g, x in zip(grads, xs)] for f, xs in ((at, grads), (lambda g: code(g.dtype), grads), (torch.Tensor.numel, params)))
            if outs is None:
                o_at, o_code = none, none
            elif _present(outs) is outs:
                o_at, o_code = map(at, outs), map(code, map(_dtype_of, outs))
            else:
                o_at, o_code = [0 if o is None else o.data_ptr() for o in outs], [0 if o is None else code(o.dtype) for o in outs]
            scales = (map(at, lists[2]), map(at, lists[3])) if eight else (none, none)
            table = _adamw_rows(n).pack(*itertools.chain.from_iterable(zip(map(at, params), g_at, map(at, lists[0]), map(at, lists[1]), *scales, o_at, count, decay,
                                                                           map(code, map(_dtype_of, params)), g_code, o_code, itertools.repeat(state.bits))))
            how = _l.AlphaAdamWStep(lr, beta1, beta2, eps, 0.0 if max_norm is None else max_norm, operator.index(step), norm_at, lr_at, step_at, seed)
            _l.check(self.base._lib.alpha_adamW(n, table, C.byref(how), _stream(self.base._stream)))
        return norm

    @staticmethod
    def _check_adamw(what, params, grads, outs, lists):
        """The GPU of a step's tensors and whether all gradients are dense; raises for tensors the library would not take.  (A pass over all tensors for each question.)"""
        T = torch.Tensor
        kept, used = [] if outs is None else _present(outs), _present(grads)
        device = params[0].get_device()
        written = params + kept
        good = (device >= 0 and set(map(T.get_device, itertools.chain(written, used, *lists))) == {device} and set(map(_dtype_of, written + used)) <= _FC_TYPES.keys()
                and all(map(T.is_contiguous, written)) and not any(map(T.is_neg, written)) and list(map(T.numel, lists[0])) == list(map(T.numel, params)))
        shapes = list(map(_shape_of, params))
        if good:
            good = list(map(_shape_of, grads)) == shapes if used is grads else all(g is None or g.shape == s for g, s in zip(grads, shapes))
        if good and outs is not None:
            good = list(map(_shape_of, outs)) == shapes if kept is outs else all(o is None or o.shape == s for o, s in zip(outs, shapes))
        if not good:
            for i, (p, g) in enumerate(zip(params, grads)):
                o = None if outs is None else outs[i]
                for name, t in (("parameter", p), ("gradient", g), ("output", o)):
                    if t is None:
                        continue
                    if t.dtype not in _FC_TYPES:
                        raise ValueError("%s: %s %d must be float32, bfloat16 or float16, not %s" % (what, name, i, t.dtype))
                    if t.shape != p.shape or t.get_device() != device or device < 0:
                        raise ValueError("%s: %s %d is %s on %s, parameter %s on %s; all belong on one GPU" % (what, name, i, tuple(t.shape), t.device, tuple(p.shape), params[0].device))
                    if t is not g and (not t.is_contiguous() or t.is_neg()):
                        raise ValueError("%s: %s %d must be dense" % (what, name, i))
                if lists[0][i].numel() != p.numel() or any(t[i].get_device() != device for t in lists):
                    raise ValueError("%s: moments %d are %s on %s, parameter %s on %s" % (what, i, tuple(lists[0][i].shape), lists[0][i].device, tuple(p.shape), p.device))
        return device, all(map(T.is_contiguous, used)) and not any(map(T.is_neg, used))

    # ---- group normalisation ----
    def groupNorm(self, X, groups, gamma=None, beta=None, eps=1e-5, act="none", k=0.0, save=False):
        """act((X - mean) / sqrt(variance + eps) * gamma + beta) of channels-last tensors X [N, ..., C] (float32, bfloat16, float16), mean and variance over the
        positions and the channels of each of `groups` groups of neighbours.  gamma, beta [C]: of X's type or float32, both or neither.  act as in fullConnect.  save=True
        also returns mean and rstd [N, groups] (float32), which groupNorm_delta reads."""
        plan = self._norm_check("groupNorm", X, operator.index(groups), gamma, beta, act, float(k), float(eps), ())
        if plan is None:
            return (X.new_empty(X.shape), _new(X, (0, groups)), _new(X, (0, groups))) if save else X.new_empty(X.shape)
        if self.base._stream is None and X.get_device() == torch._C._cuda_getDevice():
            return self._norm_run(plan, X, gamma, beta, save)
        with self._on(X):
            return self._norm_run(plan, X, gamma, beta, save)

    def _norm_run(self, plan, X, gamma, beta, save):
        shape, kept = plan
        Xd, gamma, beta = _dense_now(X), _dense_now(gamma), _dense_now(beta)
        Y = X.new_empty(X.shape)
        mean, rstd = (_new(X, kept), _new(X, kept)) if save else (None, None)
        self.base.groupNorm(shape, Xd, gamma, beta, mean, rstd, Y)
        return (Y, mean, rstd) if save else Y

    def groupNorm_delta(self, deltaY, X, mean, rstd, gamma=None, beta=None, act="none", k=0.0):
        """(deltaX, deltaGamma, deltaBeta) of groupNorm from deltaY, its X and the mean and rstd it saved; the latter two None without gamma and beta."""
        if mean.dim() != 2:
            raise ValueError("groupNorm_delta: mean %s, expected [N, groups]" % (tuple(mean.shape),))
        kept = (X.shape[0] if X.dim() else 0, mean.shape[1])
        plan = self._norm_check("groupNorm_delta", X, mean.shape[1], gamma, beta, act, float(k), 0.0,
                                (("deltaY", deltaY, X.shape, X.dtype), ("mean", mean, kept, torch.float32), ("rstd", rstd, kept, torch.float32)))
        if plan is None:
            return X.new_empty(X.shape), *(None if gamma is None else torch.zeros_like(gamma) for _ in range(2))
        if self.base._stream is None and X.get_device() == torch._C._cuda_getDevice():
            return self._norm_run_delta(plan[0], deltaY, X, mean, rstd, gamma, beta)
        with self._on(X):
            return self._norm_run_delta(plan[0], deltaY, X, mean, rstd, gamma, beta)

    def _norm_run_delta(self, shape, deltaY, X, mean, rstd, gamma, beta):
        dYd, Xd, meand, rstdd, gamma, beta = map(_dense_now, (deltaY, X, mean, rstd, gamma, beta))
        dX = X.new_empty(X.shape)
        dG, dB = (gamma.new_empty(gamma.shape), gamma.new_empty(gamma.shape)) if gamma is not None else (None, None)
        self.base.groupNorm_delta(shape, dYd, Xd, meand, rstdd, gamma, beta, dX, dG, dB)
        return dX, dG, dB

    @staticmethod
    def _norm_check(what, X, groups, gamma, beta, act, k, eps, others):
        """The checked call's plan (None where X holds nothing)."""
        if (gamma is None) != (beta is None):
            raise ValueError("%s: gamma and beta, or neither" % what)
        plan = _norm_plan(what, X.shape, groups, X.dtype, None if gamma is None else gamma.dtype, _fc_act(what, act), k, eps)
        device = X.get_device()
        if device < 0:
            raise ValueError("%s: tensors must be on a GPU" % what)
        if gamma is not None:
            others += (("gamma", gamma, X.shape[-1:], gamma.dtype), ("beta", beta, X.shape[-1:], gamma.dtype))
        for name, t, shape, dtype in others:
            if t.shape != shape:
                raise ValueError("%s: %s %s, expected %s" % (what, name, tuple(t.shape), tuple(shape)))
            if t.dtype != dtype or t.get_device() != device:
                raise ValueError("%s: %s is %s on %s, X %s on %s" % (what, name, t.dtype, t.device, X.dtype, X.device))
        return plan

    # Batched products with the engine's memory rule (only the last dimension of a tensor is padded to a multiple
    # of 4) and EngineCore's argument mapping (EngineCore.java:579-623): the row pitch and the logical row length
    # go down separately.  The batch itself is not padded here (the reference rounds it up over zero matrices).
    def batchMatMul(self, A, B):
        """C[b] = A[b] * B[b]; A [Batch, N, K], B [Batch, K, M]."""
        (Bt, N, K), (Bt2, K2, M) = A.shape, B.shape
        if Bt != Bt2 or K != K2:
            raise ValueError("batchMatMul: A %s against B %s" % (tuple(A.shape), tuple(B.shape)))
        (Ap, Bp), _held = _pad_all((A, Bt, _pad4(K)), (B, Bt, _pad4(M)))
        # the kernels write the M columns; only padding columns need zeros
        C = (torch.empty if M % 4 == 0 else torch.zeros)((Bt, N, _pad4(M)), dtype=torch.float32, device=A.device)
        self.base.batchMatMul(C, Ap, Bp, Bt, N, _pad4(M), K, _pad4(K))
        return C[..., :M]

    def batchMatMulT1(self, A, B):
        """C[b] = A[b]^T * B[b]; A [Batch, K, N], B [Batch, K, M]."""
        (Bt, K, N), (Bt2, K2, M) = A.shape, B.shape
        if Bt != Bt2 or K != K2:
            raise ValueError("batchMatMulT1: A %s against B %s" % (tuple(A.shape), tuple(B.shape)))
        (Ap, Bp), _held = _pad_all((A, Bt, _pad4(N)), (B, Bt, _pad4(M)))
        # the kernels write the M columns; only padding columns need zeros
        C = (torch.empty if M % 4 == 0 else torch.zeros)((Bt, N, _pad4(M)), dtype=torch.float32, device=A.device)
        self.base.batchMatMulT1(C, Ap, Bp, Bt, N, _pad4(N), _pad4(M), K)
        return C[..., :M]

    def batchMatMulT2(self, A, B):
        """C[b] = A[b] * B[b]^T; A [Batch, N, K], B [Batch, M, K]."""
        (Bt, N, K), (Bt2, M, K2) = A.shape, B.shape
        if Bt != Bt2 or K != K2:
            raise ValueError("batchMatMulT2: A %s against B %s" % (tuple(A.shape), tuple(B.shape)))
        (Ap, Bp), _held = _pad_all((A, Bt, _pad4(K)), (B, Bt, _pad4(K)))
        # the kernels write the M columns; only padding columns need zeros
        C = (torch.empty if M % 4 == 0 else torch.zeros)((Bt, N, _pad4(M)), dtype=torch.float32, device=A.device)
        self.base.batchMatMulT2(C, Ap, Bp, Bt, N, _pad4(M), M, _pad4(K))
        return C[..., :M]

    # ---- 2D pooling (Engine.pool2D_max / pool2D_avg and their gradients; CudaFloat32EngineBase.java:2012-2215) ----
    def _pool_shape(self, X, FH, FW, sh, sw, ph, pw):
        N, IH, IW, IC = X.shape
        OH, OW = (IH + 2 * ph - FH) // sh + 1, (IW + 2 * pw - FW) // sw + 1
        return _pool_shape(N, IH, IW, _pad4(IC), FH, FW, OH, OW, sh, sw, ph, pw), OH, OW

    def pool2D_max(self, X, FH, FW, sh, sw, ph, pw, indexed=False):
        """Y (and, with indexed=True, the int32 index tensor the indexed gradient reads)."""
        s, OH, OW = self._pool_shape(X, FH, FW, sh, sw, ph, pw)
        IC = X.shape[3]
        Xp = _pad_last(X, s.IC)
        Y = _new(X, (s.N, OH, OW, s.IC))
        if indexed:
            Index = _new(X, (s.N, OH, OW, s.IC), torch.int32)
            self.base.pool2D_max_indexed(Y, Index, OH, OW, Xp, s.IH, s.IW, FH, FW, s.N, s.IC, sh, sw, ph, pw)
            return (Y if s.IC == IC else Y[..., :IC]), Index
        self.base.pool2D_max(Y, OH, OW, Xp, s.IH, s.IW, FH, FW, s.N, s.IC, sh, sw, ph, pw)
        return Y if s.IC == IC else Y[..., :IC]

    def pool2D_avg(self, X, FH, FW, sh, sw, ph, pw, ignore_padding=False):
        s, OH, OW = self._pool_shape(X, FH, FW, sh, sw, ph, pw)
        IC = X.shape[3]
        Xp = _pad_last(X, s.IC)
        Y = _new(X, (s.N, OH, OW, s.IC))
        a = self.base._addr
        _l.check(self.base._lib.alpha_pool2D_avg(C.byref(s), a(Xp), a(Y), int(bool(ignore_padding)), _stream(self.base._stream)))
        return Y if s.IC == IC else Y[..., :IC]

    def upool2D_max(self, deltaY, Y, X, FH, FW, sh, sw, ph, pw):
        """deltaX of pool2D_max from X and Y of the forward pass."""
        s, OH, OW = self._pool_shape(X, FH, FW, sh, sw, ph, pw)
        IC = X.shape[3]
        Xp, Yp, dYp = _pad_last(X, s.IC), _pad_last(Y, s.IC), _pad_last(deltaY, s.IC)
        dX = torch.empty_like(Xp)
        a = self.base._addr
        _l.check(self.base._lib.alpha_upool2D_max(C.byref(s), a(dYp), a(Yp), a(Xp), a(dX), _stream(self.base._stream)))
        return dX if s.IC == IC else dX[..., :IC]

    def upool2D_max_indexed(self, deltaY, Index, IH, IW, FH, FW, sh, sw, ph, pw):
        """deltaX of pool2D_max from the index tensor of the forward pass (its channel count is the padded one)."""
        N, OH, OW, IC = deltaY.shape
        ic4 = Index.shape[3]
        s = _pool_shape(N, IH, IW, ic4, FH, FW, OH, OW, sh, sw, ph, pw)
        dYp = _pad_last(deltaY, ic4)
        dX = _new(deltaY, (N, IH, IW, ic4))
        a = self.base._addr
        _l.check(self.base._lib.alpha_upool2D_max_indexed(C.byref(s), a(dYp), a(Index), a(dX), _stream(self.base._stream)))
        return dX if ic4 == IC else dX[..., :IC]

    def upool2D_avg(self, deltaY, IH, IW, FH, FW, sh, sw, ph, pw, ignore_padding=False):
        N, OH, OW, IC = deltaY.shape
        ic4 = _pad4(IC)
        s = _pool_shape(N, IH, IW, ic4, FH, FW, OH, OW, sh, sw, ph, pw)
        dYp = _pad_last(deltaY, ic4)
        dX = _new(deltaY, (N, IH, IW, ic4))
        a = self.base._addr
        _l.check(self.base._lib.alpha_upool2D_avg(C.byref(s), a(dYp), a(dX), int(bool(ignore_padding)), _stream(self.base._stream)))
        return dX if ic4 == IC else dX[..., :IC]

    def dconv3D(self, X, W, sh, sw, ph, pw, OH=None, OW=None):
        """Deconv3D forward = dconv3D_deltaX with the roles of input and output swapped
        (Engine.java:1819-1829); W is [IC_in, FH, FW, OC_out]."""
        N, IH, IW, _ = X.shape
        _, FH, FW, _ = W.shape
        if OH is None:
            OH = (IH - 1) * sh + FH - 2 * ph
        if OW is None:
            OW = (IW - 1) * sw + FW - 2 * pw
        return self.dconv3D_deltaX(X, W, OH, OW, sh, sw, ph, pw)
