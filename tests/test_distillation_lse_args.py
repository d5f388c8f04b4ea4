"""The C entry point of the distillation with a float64 teacher_lse: what it refuses before any launch.  No GPU."""
import ctypes

from test_logits_args import EDTYPE, EINVAL, EWORKSPACE, FAKE, F64, distill_desc, i64, lib, vp  # noqa: F401


def test_refusals(lib):  # noqa: F811
    fwd, ref = lib.supa_amd_distill_forward_lse64, ctypes.byref
    need = lib.supa_amd_distill_workspace_bytes(ref(distill_desc()))

    def forward(d=None, lse=FAKE, loss=FAKE, count=FAKE, stats=FAKE, ws=FAKE, size=need):
        d = distill_desc() if d is None else d
        return fwd(ref(d), vp(lse), vp(loss), vp(count), vp(stats), None, vp(ws), i64(size), None, None)

    assert fwd(None, vp(FAKE), vp(FAKE), vp(FAKE), vp(FAKE), None, vp(FAKE), i64(need), None, None) == EINVAL
    assert forward(lse=None) == EINVAL and forward(distill_desc(teacher_lse=FAKE), lse=None) == EINVAL
    assert forward(loss=None) == EINVAL and forward(count=None) == EINVAL and forward(stats=None) == EINVAL
    assert forward(ws=None) == EWORKSPACE and forward(size=need - 1) == EWORKSPACE and forward(ws=FAKE + 4) == EINVAL
    assert forward(distill_desc(dtype=F64)) == EDTYPE and forward(distill_desc(temperature=0.0)) == EINVAL
    assert forward(distill_desc(rows=0, reduction=0), lse=None) == 0
