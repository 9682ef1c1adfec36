"""Microscaled storage on the device: tensors in 8 or 4 bits with one power-of-two scale per 32 channels (include/msc.h, msc_mx_*).

The reference trains and serves in float32 and has no counterpart; these stand beside the engine's 16-bit operators:

  pack / unpack        a tensor to E4M3 (one byte per element) or E2M1 (half a byte) and back; beside msc_pack_cast
  conv_weight_grad     weight gradient of a convolution / linear layer from the E4M3 checkpoint of its input; beside msc_conv_wgrad
  batchnorm_backward   BatchNorm (+ ReLU, + residual join) backward from the E4M3 checkpoint of its input; beside msc_bn_bwd_reduce / _apply
  linear               a pointwise convolution / linear layer on E2M1 operands, for serving; beside the 1x1 form of msc_conv_igemm

Tensors are [..., C], a row of channels per pixel or token: NHWC activations, a channel slice of one, or [rows, C].  float32, bfloat16 and float16.
Calls run on the current stream of the tensors' device, take their scratch from torch's allocator, never synchronise and may be captured into a
hipGraph; results are the same bits from run to run.  Nothing is recorded by autograd.

A training step that keeps its activations in 8 bits calls pack behind each layer's forward and conv_weight_grad / batchnorm_backward in its backward:
UNetResNet(activation_checkpoint='e4m3') does so.
"""
import ctypes as C

import torch

from . import _lib

FORMATS = {'e4m3': (_lib.MX_E4M3, 32), 'e2m1': (_lib.MX_E2M1, 16)}       # name -> (id, bytes of a block's codes)
_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


class MxTensor:
    """A packed tensor of shape [..., channels]: codes uint8 [..., blocks * 32 (E4M3) or 16 (E2M1)], scales uint8 [..., blocks], blocks = ceil(channels / 32).
    Rows of codes start on 16 bytes; both may be slices of wider buffers.
    dtype: the type of the tensor that was packed (pack sets it), or None where the codes come from elsewhere and nobody said.  The values depend on codes and scales alone; the
    type says which numbers they can be (conv_weight_grad)."""
    __slots__ = ('_codes', '_scales', '_buf', '_lead', 'channels', 'fmt', 'dtype')

    def __init__(self, codes, scales, channels, fmt='e4m3', dtype=None):
        if fmt not in FORMATS:
            raise ValueError("format must be 'e4m3' or 'e2m1', got %r" % (fmt,))
        if dtype is not None and dtype not in _DTYPES:
            raise TypeError('a packed tensor was float32, bfloat16 or float16, got %s' % (dtype,))
        nb = (channels + 31) // 32
        if channels <= 0 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError('a packed tensor has at least one channel, and uint8 codes and scales')
        lead = codes.shape[:-1]
        if codes.shape[-1] != nb * FORMATS[fmt][1] or scales.shape[-1] != nb or lead != scales.shape[:-1]:
            raise ValueError('%d channels in %s take %d code bytes and %d scales per row, got codes %s and scales %s'
                             % (channels, fmt, nb * FORMATS[fmt][1], nb, tuple(codes.shape), tuple(scales.shape)))
        if codes.device != scales.device:
            raise ValueError('codes and scales are on different devices')
        self._codes, self._scales, self._buf, self._lead, self.channels, self.fmt, self.dtype = codes, scales, None, lead, channels, fmt, dtype

    @classmethod
    def _made(cls, buf, lead, channels, fmt, dtype=None):
        """over one allocation, the codes and then the scales; the two tensors are made when somebody asks for them (each costs the host what a launch does)"""
        t = cls.__new__(cls)
        t._codes, t._scales, t._buf, t._lead, t.channels, t.fmt, t.dtype = None, None, buf, lead, channels, fmt, dtype
        return t

    def _split(self):
        nb, per = (self.channels + 31) // 32, FORMATS[self.fmt][1]
        n = self._buf.numel() // (per + 1) * per
        self._codes, self._scales = self._buf[:n].view(self._lead + (nb * per,)), self._buf[n:].view(self._lead + (nb,))

    @property
    def codes(self):
        if self._codes is None:
            self._split()
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            self._split()
        return self._scales

    @property
    def shape(self):
        return self._lead + (self.channels,)

    @property
    def device(self):
        return (self._codes if self._buf is None else self._buf).device

    @property
    def nbytes(self):
        return self._codes.numel() + self._scales.numel() if self._buf is None else self._buf.numel()

    def _args(self, what):
        """rows, address and row pitch of the codes, of the scales"""
        buf = self._buf
        if buf is None:
            codes, scales = self._codes, self._scales
            rows, c_ld = _rows(codes, what)
            return rows, codes.data_ptr(), c_ld, scales.data_ptr(), _rows(scales, what)[1]
        if not buf.is_cuda:
            raise _lib.MscError('%s: needs a CUDA/ROCm tensor; there is no CPU path in the product' % what)
        nb, per = (self.channels + 31) // 32, FORMATS[self.fmt][1]
        rows, at = buf.numel() // (nb * (per + 1)), buf.data_ptr()
        return rows, at, nb * per, at + rows * nb * per, nb


def _rows(t, what):
    """(rows, elements from row to row) of a tensor [..., C] whose rows are equally far apart"""
    if not t.is_cuda:
        raise _lib.MscError('%s: needs a CUDA/ROCm tensor; there is no CPU path in the product' % what)
    if t.dim() < 2:
        raise ValueError('%s: expected [..., channels], got shape %s' % (what, tuple(t.shape)))
    shape = t.shape
    if t.is_contiguous():
        return t.numel() // shape[-1] if shape[-1] else 0, shape[-1]
    stride = t.stride()
    if shape[-1] > 1 and stride[-1] != 1:
        raise ValueError('%s: channels have to be next to each other (strides %s)' % (what, tuple(stride)))
    pitch, rows = None, 1
    for n, s in zip(reversed(shape[:-1]), reversed(stride[:-1])):
        if n != 1:
            if pitch is None:
                pitch = s
            elif s != pitch * rows:
                raise ValueError('%s: expected an NHWC tensor or a channel slice of one (shape %s, strides %s)' % (what, tuple(shape), tuple(stride)))
        rows *= n
    return rows, max(shape[-1], 1) if pitch is None or rows == 0 else pitch


def _dtype(t, what):
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError('%s: float32, bfloat16 or float16, got %s' % (what, t.dtype)) from None


def _same_device(what, dev, *ts):
    for t in ts:
        if t is not None and t.device != dev:
            raise ValueError('%s: tensors on %s and %s' % (what, dev, t.device))


def _vector(t, n, dev, what):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous() or t.device != dev:
        raise ValueError('%s: expected %d contiguous float32 values on %s' % (what, n, dev))
    return t.data_ptr()


def _out(out, shape, dtype, dev, what):
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != dev:
        raise ValueError('%s: out has to be %s %s on %s' % (what, tuple(shape), dtype, dev))
    return out


# Small calls are bound by the host (a launch costs it 3 us, an allocation 1.1-1.7): hence the bound entries, the stream's handle alone (the Stream object that
# torch.cuda.current_stream() makes costs 2 us), and empty_like where a result has an operand's shape.
_entries = {}


def _entry(name):
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    return fn


def _run(name, dev, *args):
    """one C call on `dev`'s current stream, with `dev` current"""
    fn, index = _entry(name), dev.index
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, name)


def _workspace(nbytes, dev, name):
    """scratch of one call; None where it needs none"""
    if nbytes < 0:
        _lib.check(-1, name)
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _new(like, shape, contiguous):
    """an uninitialised tensor of like's type and device; contiguous: `like` is, and has this shape"""
    return torch.empty_like(like) if contiguous else like.new_empty(shape)


def empty(shape, fmt='e4m3', device='cuda'):
    """an uninitialised MxTensor of `shape` [..., channels]"""
    lead, c = torch.Size(shape[:-1]), shape[-1]
    if fmt not in FORMATS:
        raise ValueError("format must be 'e4m3' or 'e2m1', got %r" % (fmt,))
    if c <= 0:
        raise ValueError('a packed tensor has at least one channel')
    return MxTensor._made(torch.empty(lead.numel() * ((c + 31) // 32) * (FORMATS[fmt][1] + 1), dtype=torch.uint8, device=device), lead, c, fmt)


def pack(x, fmt='e4m3', out=None):
    """x [..., C] in blocks of 32 channels: the smallest power-of-two scale under which nothing passes the largest code, then the nearest code (ties to
    even).  A block that holds an infinity or NaN stands for 32 NaNs.  Returns an MxTensor (`out`, if given)."""
    if fmt not in FORMATS:
        raise ValueError("format must be 'e4m3' or 'e2m1', got %r" % (fmt,))
    rows, ld = _rows(x, 'pack')
    shape, dev = x.shape, x.device
    c, (fid, per) = shape[-1], FORMATS[fmt]
    if out is None:
        if c <= 0:
            raise ValueError('a packed tensor has at least one channel')
        nb = (c + 31) // 32
        buf = torch.empty(rows * nb * (per + 1), dtype=torch.uint8, device=dev)
        out = MxTensor._made(buf, shape[:-1], c, fmt)
        cp, c_ld, s_ld = buf.data_ptr(), nb * per, nb
        sp = cp + rows * c_ld
    else:
        if out.shape != shape or out.fmt != fmt:
            raise ValueError('pack: out holds %s in %s, not %s in %s' % (tuple(out.shape), out.fmt, tuple(shape), fmt))
        _same_device('pack', dev, out)
        _, cp, c_ld, sp, s_ld = out._args('pack')
    _run('msc_mx_pack', dev, x.data_ptr(), ld, _dtype(x, 'pack'), cp, c_ld, sp, s_ld, fid, rows, c)
    out.dtype = x.dtype
    return out


def unpack(t, dtype=torch.bfloat16, out=None):
    """the values an MxTensor stands for, in `dtype` (any of the three; the one that was packed holds every value exactly)"""
    rows, cp, c_ld, sp, s_ld = t._args('unpack')
    dev, c = t.device, t.channels
    if out is None:
        out, ld = torch.empty(t._lead + (c,), dtype=dtype, device=dev), c
    else:
        _out(out, t.shape, out.dtype, dev, 'unpack')
        ld = _rows(out, 'unpack')[1]
    _run('msc_mx_unpack', dev, cp, c_ld, sp, s_ld, FORMATS[t.fmt][0], out.data_ptr(), ld, _dtype(out, 'unpack'), rows, c)
    return out


def conv_weight_grad(dy, saved, kernel=1, stride=1, pad=0, out=None, accumulate=False):
    """float32 [A, KH, KW, B]: the weight gradient of a convolution whose output gradient is dy [N, H, W, A] and whose input [N, Hi, Wi, B] was kept as the E4M3
    MxTensor `saved`.  kernel: a size or (KH, KW).  A linear layer: kernel 1, dy [..., A] and saved [..., B] with the same leading shape.
    accumulate: added to `out` (which then has to be given) instead of written over it.
    The products are of dy's type, in which every value of a checkpoint of that type is exact.  float16 does not hold every value of a wider one (past 65504, below 2^-24): a
    float16 dy with a checkpoint that was packed from float32 or bfloat16 (saved.dtype) is turned to float32 first.  saved.dtype None: taken to be dy's."""
    if saved.fmt != 'e4m3':
        raise ValueError('conv_weight_grad: the checkpoint has to be in e4m3, got %s' % saved.fmt)
    if accumulate and out is None:
        raise ValueError('conv_weight_grad: accumulate needs out')
    kh, kw = (kernel, kernel) if isinstance(kernel, int) else kernel
    if dy.dtype == torch.float16 and saved.dtype not in (None, torch.float16):
        dy = dy.float()
    rows, p_ld = _rows(dy, 'conv_weight_grad')
    _, qp, q_ld, sp, s_ld = saved._args('conv_weight_grad')
    a, b = dy.shape[-1], saved.channels
    if kh == 1 and kw == 1 and stride == 1 and pad == 0:
        if dy.shape[:-1] != saved._lead:
            raise ValueError('conv_weight_grad: dy %s and input %s differ in their rows' % (tuple(dy.shape), tuple(saved.shape)))
        n, hp, wp, hq, wq = rows, 1, 1, 1, 1
    else:
        if dy.dim() != 4 or len(saved.shape) != 4 or dy.shape[0] != saved.shape[0]:
            raise ValueError('conv_weight_grad: expected NHWC dy and input, got %s and %s' % (tuple(dy.shape), tuple(saved.shape)))
        (n, hp, wp), (hq, wq) = dy.shape[:3], saved.shape[1:3]
        want = tuple((i + 2 * pad - k) // stride + 1 if stride > 0 else 0 for i, k in ((hq, kh), (wq, kw)))
        if (hp, wp) != want:
            raise ValueError('conv_weight_grad: an input of %dx%d gives an output of %dx%d, dy is %dx%d' % (hq, wq, want[0], want[1], hp, wp))
    dev = dy.device
    if out is None:
        out = torch.empty((a, kh, kw, b), dtype=torch.float32, device=dev)
    elif not _out(out, (a, kh, kw, b), torch.float32, dev, 'conv_weight_grad').is_contiguous():
        raise ValueError('conv_weight_grad: out has to be contiguous')
    _same_device('conv_weight_grad', dev, saved)
    d = _lib.MxWgradDesc(dy.data_ptr(), qp, sp, out.data_ptr(), None, p_ld, q_ld, s_ld, _dtype(dy, 'conv_weight_grad'),
                         n, hp, wp, a, hq, wq, b, kh, kw, stride, pad, accumulate)
    ref = C.byref(d)
    ws = _workspace(_entry('msc_mx_wgrad_workspace_bytes')(ref), dev, 'msc_mx_wgrad_workspace_bytes')
    if ws is not None:
        d.ws = ws.data_ptr()
    _run('msc_mx_wgrad', dev, ref)
    return out


def batchnorm_backward(dout, saved, gamma, mean, invstd, relu_mask=None, scale=None, shift=None, residual=False, dy=None):
    """Backward of out = relu?(batchnorm(y) (+ res)) in training mode, with y [..., C] kept as the E4M3 MxTensor `saved` and mean / invstd the forward's
    batch statistics: (dy, dgamma, dbeta) or, with residual, (dy, dgamma, dbeta, dres).
    The ReLU: relu_mask, the byte mask msc_bn_apply writes ([..., ceil(C / 8)], for float32 ceil(C / 4)); or scale and shift, the forward's coefficients, from
    which the mask is recomputed on the stored y; or neither: no ReLU.  gamma may be None (ones).  dy may be dout (in place)."""
    if saved.fmt != 'e4m3':
        raise ValueError('batchnorm_backward: the checkpoint has to be in e4m3, got %s' % saved.fmt)
    if dout.shape != saved.shape:
        raise ValueError('batchnorm_backward: dout %s and input %s differ' % (tuple(dout.shape), tuple(saved.shape)))
    if (scale is None) != (shift is None) or (scale is not None and relu_mask is not None):
        raise ValueError('batchnorm_backward: the ReLU takes relu_mask, or scale and shift, or neither')
    dev, c = dout.device, saved.channels
    rows, dout_ld = _rows(dout, 'batchnorm_backward')
    _, yp, y_ld, sp, s_ld = saved._args('batchnorm_backward')
    _same_device('batchnorm_backward', dev, saved, relu_mask)
    dt, dtype, dense = _dtype(dout, 'batchnorm_backward'), dout.dtype, dout.is_contiguous()
    relu, mask_ld = 0, 0
    if relu_mask is not None:
        per = 4 if dt == _lib.F32 else 8
        if relu_mask.dtype != torch.uint8 or relu_mask.shape != dout.shape[:-1] + ((c + per - 1) // per,):
            raise ValueError('batchnorm_backward: the mask has one byte for %d channels of a row, got %s %s' % (per, tuple(relu_mask.shape), relu_mask.dtype))
        relu, mask_ld = 3, _rows(relu_mask, 'batchnorm_backward')[1]
    elif scale is not None:
        relu = 2
    if dy is None:
        dy, dy_ld = _new(dout, dout.shape, dense), c
    else:
        dy_ld = _rows(_out(dy, dout.shape, dtype, dev, 'batchnorm_backward'), 'batchnorm_backward')[1]
    mean_p = _vector(mean, c, dev, 'batchnorm_backward: mean')
    dgamma, dbeta = _new(mean, (c,), mean.dim() == 1), _new(mean, (c,), mean.dim() == 1)
    dres = _new(dout, dout.shape, dense) if residual else None
    ws = _workspace(_entry('msc_mx_bn_bwd_workspace_bytes')(rows, c), dev, 'msc_mx_bn_bwd_workspace_bytes')
    d = _lib.MxBnBwdDesc(dout.data_ptr(), yp, sp, relu_mask.data_ptr() if relu_mask is not None else None,
                         _vector(gamma, c, dev, 'batchnorm_backward: gamma'), mean_p,
                         _vector(invstd, c, dev, 'batchnorm_backward: invstd'), _vector(scale, c, dev, 'batchnorm_backward: scale'),
                         _vector(shift, c, dev, 'batchnorm_backward: shift'), dgamma.data_ptr(), dbeta.data_ptr(), dy.data_ptr(),
                         dres.data_ptr() if residual else None, ws.data_ptr() if ws is not None else None, dout_ld, y_ld, s_ld, mask_ld, dy_ld, c, rows,
                         dt, c, relu, 0, 0)
    _run('msc_mx_bn_bwd', dev, C.byref(d))
    return (dy, dgamma, dbeta, dres) if residual else (dy, dgamma, dbeta)


def linear(x, w, scale=None, shift=None, res=None, relu=False, dtype=None, out=None):
    """act(scale * (x @ w.T) + shift + res) [..., N]: x [..., K] a tensor (quantised to E2M1 within the call) or an E2M1 MxTensor (dtype: the result's,
    bfloat16 if not given), w the E2M1 MxTensor of a weight [N, K]; scale / shift float32 [N] (a folded BatchNorm, a bias), res [..., N] in the result's
    dtype.  out may be res."""
    packed = isinstance(x, MxTensor)
    if w.fmt != 'e2m1' or (packed and x.fmt != 'e2m1'):
        raise ValueError('linear: the operands have to be in e2m1')
    k = w.channels
    if len(w._lead) != 1 or k != x.shape[-1]:
        raise ValueError('linear: x %s and w %s do not go together' % (tuple(x.shape), tuple(w.shape)))
    dev, (n,) = x.device, w._lead
    if dtype is None:
        dtype = x.dtype if not packed else out.dtype if out is not None else res.dtype if res is not None else torch.bfloat16
    if not packed and x.dtype != dtype:
        raise ValueError('linear: the result has the type of x')
    if packed:
        m, xcp, xc_ld, xsp, xs_ld = x._args('linear')
        xp, x_ld = None, 0
    else:
        m, x_ld = _rows(x, 'linear')
        xp, xcp, xsp, xc_ld, xs_ld = x.data_ptr(), None, None, 0, 0
    shape = x.shape[:-1] + (n,)
    if out is None:
        out, out_ld = torch.empty(shape, dtype=dtype, device=dev) if packed else x.new_empty(shape), n
    else:
        out_ld = _rows(_out(out, shape, dtype, dev, 'linear'), 'linear')[1]
    _same_device('linear', dev, w)
    resp, res_ld = (None, 0) if res is None else (res.data_ptr(), _rows(_out(res, shape, dtype, dev, 'linear: res'), 'linear')[1])
    if m == 0:
        return out
    _, wp, w_ld, wsp, ws_ld = w._args('linear')
    d = _lib.MxLinearDesc(xp, xcp, xsp, wp, wsp, _vector(scale, n, dev, 'linear: scale'), _vector(shift, n, dev, 'linear: shift'), resp,
                          out.data_ptr(), None, x_ld, xc_ld, xs_ld, w_ld, ws_ld, res_ld, out_ld, m,
                          _dtype(out, 'linear'), k, n, relu)
    ref = C.byref(d)
    ws = _workspace(_entry('msc_mx_linear_workspace_bytes')(ref), dev, 'msc_mx_linear_workspace_bytes')
    if ws is not None:
        d.ws = ws.data_ptr()
    _run('msc_mx_linear', dev, ref)
    return out
