"""Runs under FLODL_B200_BOUNDS_CHECK=1 (the debug library): attention over another sequence records nothing over ragged shapes and masks, and lists of live blocks that
say what cannot be are recorded as {site, index, limit}, with the block left out and the context intact."""
import ctypes
import math
import os
import sys

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [os.path.dirname(HERE), HERE]
from flodl_b200 import _ext, ops  # noqa: E402
from test_attention_c_entries_cpu import Cross  # noqa: E402

C = _ext.require()
assert C.bounds_check_build(), "this worker needs the bounds-checked library"
C.bounds_report(True)


def normal(*s):
    return torch.randn(*s, device="cuda").bfloat16()


for B, Sq, Sk, H, Hk, D in ((2, 3, 40, 2, 2, 64), (2, 130, 300, 4, 2, 128), (24, 130, 300, 16, 16, 64), (2, 400, 9000, 2, 1, 64), (70, 17, 600, 8, 8, 64), (300, 3, 30, 2, 2, 64)):
    leaves = [t.requires_grad_() for t in (normal(B, Sq, H, D), normal(B, Sk, Hk, D), normal(B, Sk, Hk, D))]
    mask = torch.rand(B, Sk, device="cuda") < 0.3
    mask[0, :Sk // 2] = False
    mask[-1] = False
    for m in (None, mask):
        o = ops.cross_attention(*leaves, m)
        torch.autograd.grad(o, leaves, torch.randn_like(o))
assert C.bounds_report(True) == [0, 0, 0], "what the kernels hand to one another must leave the record empty"

# ---- a list from the forward pass, spoiled before the backward pass reads it
lib = ctypes.CDLL(C.__file__)
lib.fb_cross_workspace.restype = lib.fb_cross_mask_info.restype = ctypes.c_longlong
B, Sq, Sk, H, D = 2, 5, 300, 2, 64
t = {n: normal(B, s, H, D) for n, s in (("q", Sq), ("k", Sk), ("v", Sk), ("d_o", Sq), ("o", Sq), ("dq", Sq), ("dk", Sk), ("dv", Sk))}
mask = torch.ones(B, Sk, dtype=torch.bool, device="cuda")
stats = torch.zeros(B * H * Sq, device="cuda")
a = Cross(B=B, H=H, Hk=H, Sq=Sq, Sk=Sk, D=D, scale=1 / math.sqrt(D), mask=mask.data_ptr(), mask_stride=Sk, mask_bool=1, stats=stats.data_ptr(),
          **{n: v.data_ptr() for n, v in t.items()})
for n in ("q", "k", "v", "o", "do", "dq", "dk"):
    getattr(a, n + "_strides")[:] = t["d_o" if n == "do" else n].stride()[:3]
info = torch.zeros(lib.fb_cross_mask_info(ctypes.byref(a)), dtype=torch.int32, device="cuda")
space = torch.zeros(max(lib.fb_cross_workspace(ctypes.byref(a), b) for b in (0, 1)), device="cuda")
a.mask_info, a.workspace = info.data_ptr(), space.data_ptr()
torch.cuda.synchronize()
assert lib.fb_cross_attn_fwd(ctypes.byref(a), None) == 0
torch.cuda.synchronize()
assert info[:B].tolist() == [3, 3] and info[2 * B:].tolist() == [0, 2, 5] * 2        # counts; block << 1 | by the table, as the last one is
for at, value, site, index, limit in ((2 * B + 1, 500 << 1, 302, 500, 3), (0, 9, 301, 9, 4)):
    kept = info.clone()
    info[at] = value
    torch.cuda.synchronize()
    assert lib.fb_cross_attn_bwd(ctypes.byref(a), None) == 0
    record = C.bounds_report(True)
    assert tuple(record) == (site, index, limit), record
    info.copy_(kept)
assert lib.fb_cross_attn_bwd(ctypes.byref(a), None) == 0 and C.bounds_report(True) == [0, 0, 0]
assert torch.ones(4, device="cuda").sum().item() == 4.0      # the context is still usable
print("BOUNDS_OK")
