"""CPU: the C-ABI library loads, exports every symbol include/od_boxes.h declares, and rejects bad
arguments with error codes before anything touches a GPU."""
import ctypes
import os
import re

import pytest
import torch

from object_detection_amd import _C

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _declared_symbols():
    text = open(os.path.join(ROOT, "include", "od_boxes.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(od_[a-z_0-9]+)\s*\(", text)))


def test_header_symbols_exported_and_bound():
    lib = _C.lib()
    names = _declared_symbols()
    assert len(names) >= 14
    for n in names:
        assert hasattr(lib, n), f"{n} declared in include/od_boxes.h but not exported"
        assert n in _C.SIGNATURES, f"{n} has no ctypes prototype"
    assert sorted(_C.SIGNATURES) == names
    assert lib.od_version() >= 100


def test_header_constants_match_python():
    text = open(os.path.join(ROOT, "include", "od_boxes.h")).read()
    defs = dict(re.findall(r"#define\s+(OD_[A-Z_0-9]+)\s+\(?(-?\d+)\)?", text))
    assert int(defs["OD_MAX_LEVELS"]) == _C.OD_MAX_LEVELS
    assert int(defs["OD_MAX_TOPK"]) == _C.OD_MAX_TOPK
    assert int(defs["OD_MAX_NMS_BOXES"]) == _C.OD_MAX_NMS_BOXES
    assert int(defs["OD_NMS_AUTO_GPU"]) == _C.NMS_AUTO_GPU and int(defs["OD_CODER_LINEAR"]) == _C.CODER_LINEAR
    assert int(defs["OD_KERNEL_COUNT"]) == len(_C.KERNEL_NAMES)


def test_workspace_sizes_host_only():
    lib = _C.lib()
    assert lib.od_match_retinanet_workspace_bytes(2000, 64, 786240) >= 2000 * 4 + 64 * 786240 * 4
    assert lib.od_matcher_workspace_bytes(10, 100) >= 40
    sizes = (ctypes.c_int64 * 2)(1000, 10)
    nbytes = lib.od_select_candidates_workspace_bytes(sizes, 2, 3, 4)
    assert nbytes >= 3 * 4040 * 8
    assert lib.od_select_candidates_workspace_bytes(sizes, 99, 3, 4) == 0       # too many levels
    assert lib.od_batched_nms_workspace_bytes(2, 6, 1000) >= 3 * 2 * 6000 * 4
    assert lib.od_batched_nms_workspace_bytes(2, 6, 5000) >= 3 * 2 * 30000 * 4  # topk_candidates = 5000 on six levels
    assert lib.od_batched_nms_workspace_bytes(2, 8, 8193) == 0                  # beyond OD_MAX_NMS_BOXES
    assert lib.od_batched_nms_workspace_bytes(2, 65, 10) == 0                   # too many segments


def test_argument_errors_without_gpu():
    lib = _C.lib()
    null = ctypes.c_void_p(0)
    i32 = (ctypes.c_int32 * 1)(4)
    assert lib.od_anchor_generate(null, null, null, null, null, null, 1, null, 0, null) == -1
    assert lib.od_anchor_generate(i32, i32, i32, i32, i32, (ctypes.c_float * 64)(), 9, ctypes.c_void_p(16), 0, null) == -2
    assert lib.od_match_retinanet(null, 0, 10, null, null, 0, 1, 0.6, 0.5, 1, null, null, 0, null) == -1
    import ctypes as ct
    bad = (ct.c_int64 * 6)(0, 64, 4, 128, 64, 4)                     # second grid starts inside the first
    assert lib.od_match_retinanet_grids(null, 0, 1024, bad, 2, null, null, 0, 1, 0.6, 0.5, 1, null, null, 0, null) == -1
    beyond = (ct.c_int64 * 3)(512, 64, 16)                           # reaches past the last anchor
    assert lib.od_match_retinanet_grids(null, 0, 1024, beyond, 1, null, null, 0, 1, 0.6, 0.5, 1, null, null, 0, null) == -1
    assert lib.od_matcher(null, 0, 5, 0.6, 0.5, 1, null, null, 0, null) == -1
    assert lib.od_batched_nms(null, null, null, null, 1, 10, 0, 1, 0.5, 0, 10, null, null, null, null, null, null, 0, null) == -1
    assert lib.od_batched_nms(ctypes.c_void_p(16), ctypes.c_void_p(16), null, ctypes.c_void_p(16), 1, 70000, 0, 1, 0.5, 0,
                              10, null, ctypes.c_void_p(16), ctypes.c_void_p(16), null, ctypes.c_void_p(16),
                              ctypes.c_void_p(256), 1 << 30, null) == -2
    # the no-allocation variant rejects sizes beyond its built-in scratch array before anything touches a GPU
    assert lib.od_batched_nms_noalloc(null, null, null, null, 8, 8192, 1, 64, 0.5, 0, 10, null, null, null, null, null,
                                      null) == -2
    assert lib.od_batched_nms_noalloc(null, null, null, null, 0, 10, 0, 1, 0.5, 0, 10, null, null, null, null, null,
                                      null) == -1
    assert lib.od_profile_select(99) == -1
    with pytest.raises(_C.OdBoxesError):
        _C.check(-3, "x")


def test_argument_errors_of_loss_transform_and_planar_entries():
    """The entry points added for the head losses, the input transform and the channel-major selection reject bad
    arguments before anything is launched (no GPU needed)."""
    lib = _C.lib()
    null, p16, p256 = ctypes.c_void_p(0), ctypes.c_void_p(16), ctypes.c_void_p(256)
    assert lib.od_focal_loss_workspace_bytes(786240, 4, 16) >= 16 * 768 * 12
    assert lib.od_focal_loss_workspace_bytes(-1, 4, 16) == 0
    # unknown element type, null logits, workspace too small
    assert lib.od_focal_loss_forward(p16, 7, 40, 10, 4, p16, p16, p16, 1, 0.25, 2.0, 0, p16, p16, p16, p256, 1 << 20, null) == -1
    assert lib.od_focal_loss_forward(null, 0, 40, 10, 4, p16, p16, p16, 1, 0.25, 2.0, 0, p16, p16, p16, p256, 1 << 20, null) == -1
    assert lib.od_focal_loss_forward(p16, 0, 40, 10, 4, p16, p16, p16, 1, 0.25, 2.0, 5, p16, p16, p16, p256, 1 << 20, null) == -1
    assert lib.od_focal_loss_forward(p16, 0, 40, 10, 4, p16, p16, p16, 1, 0.25, 2.0, 1, p16, p16, p16, p256, 8, null) == -3
    assert lib.od_focal_loss_backward(p16, 1, 40, 10, 4, p16, p16, p16, 1, 0.25, 2.0, 0, null, p16, p16, null) == -1
    assert lib.od_fcos_box_loss_forward(p16, null, 0, 40, 10, p16, 0, 10, p16, p16, p16, 1, 1e-7, p16, p16, p16, p256,
                                        1 << 20, null) == -1                          # centre-ness missing
    w = (ctypes.c_float * 4)(1.0, 1.0, 1.0, 1.0)
    zero_w = (ctypes.c_float * 4)(1.0, 0.0, 1.0, 1.0)
    assert lib.od_box_loss_workspace_bytes(1000, 2) > 0
    assert lib.od_box_loss_forward(p16, 0, 40, p16, 0, 10, p16, p16, p16, 1, 9, 1.0, w, 4.135, 1e-7, p16, p16, p16, p256,
                                   1 << 20, null) == -1                               # unknown loss type
    assert lib.od_box_loss_forward(p16, 0, 40, p16, 0, 10, p16, p16, p16, 1, 2, 1.0, zero_w, 4.135, 1e-7, p16, p16, p16,
                                   p256, 1 << 20, null) == -1                         # a zero coder weight
    assert lib.od_box_loss_forward(ctypes.c_void_p(20), 0, 40, p16, 0, 10, p16, p16, p16, 1, 2, 1.0, w, 4.135, 1e-7, p16,
                                   p16, p16, p256, 1 << 20, null) == -1               # rows not aligned to four elements
    imgs = (ctypes.c_void_p * 1)(16)
    one = (ctypes.c_int32 * 1)(8)
    big = (ctypes.c_int32 * 1)(64)
    f3 = (ctypes.c_float * 5)(0.5, 0.5, 0.5, 0.5, 0.5)
    assert lib.od_preprocess_images(imgs, one, one, one, one, 1, 5, f3, f3, p16, 32, 32, null) == -1    # > 4 channels
    assert lib.od_preprocess_images(imgs, one, one, big, one, 1, 3, f3, f3, p16, 32, 32, null) == -1    # resized > batch
    assert lib.od_preprocess_images(imgs, one, one, one, one, 0, 3, f3, f3, p16, 32, 32, null) == 0     # empty batch
    sizes = (ctypes.c_int64 * 1)(90)
    ptrs = (ctypes.c_void_p * 1)(16)
    strides = (ctypes.c_int64 * 1)(360)
    args = (ptrs, strides, None, None, ptrs, strides, ptrs, (ctypes.c_int64 * 1)(0), sizes)
    tail = (1, 1, 4, p16, 0.5, 10, 0, 4.135, p16, p16, p16, null, p16, p256, 1 << 20, null)
    assert lib.od_select_candidates_planar(*args, None, *tail) == -1                  # plane sizes missing
    assert lib.od_select_candidates_planar(*args, (ctypes.c_int64 * 1)(7), *tail) == -1   # 90 anchors are not a multiple of 7
    assert lib.od_profile_stride(0) == -1 and lib.od_profile_stride(1) == 0
    # message of the detections all-gather: negative sizes, null pointers, misaligned boxes, empty batch
    assert lib.od_pack_detections(p16, p16, p16, p16, -1, 10, p16, null) == -1
    assert lib.od_pack_detections(null, p16, p16, p16, 2, 10, p16, null) == -1
    assert lib.od_pack_detections(ctypes.c_void_p(20), p16, p16, p16, 2, 10, p16, null) == -1
    assert lib.od_pack_detections(p16, p16, p16, p16, 70000, 10, p16, null) == -2
    assert lib.od_pack_detections(null, null, null, null, 0, 10, null, null) == 0


def test_no_cpu_fallback():
    from object_detection_amd import boxes, kernels
    with pytest.raises(RuntimeError, match="GPU tensor"):
        kernels.box_iou(torch.zeros((1, 4)), torch.zeros((1, 4)))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        boxes.nms(torch.zeros((2, 4)), torch.zeros(2), 0.5)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        kernels.match_retinanet(torch.zeros((4, 4)), [torch.zeros((1, 4))], 0.6, 0.5)


def test_argument_errors_of_group_norm_act():
    lib = _C.lib()
    null, p16, p256 = ctypes.c_void_p(0), ctypes.c_void_p(16), ctypes.c_void_p(256)
    size = lib.od_group_norm_act_workspace_bytes(16, 65536, 256, 32)
    assert size >= 16 * 256 * 8
    assert lib.od_group_norm_act_workspace_bytes(1, 64, 256, 3) == 0            # groups do not divide the channels
    assert lib.od_group_norm_act_workspace_bytes(1, 64, 4096, 32) == 0          # channel limit
    assert lib.od_group_norm_act_workspace_bytes(70000, 64, 256, 32) == 0       # batch limit

    def fwd(x=p256, dtype=0, batch=2, pixels=64, channels=32, groups=4, pdtype=0, act=1, y=p256, ws=p256, nbytes=1 << 20):
        return lib.od_group_norm_act_forward(x, dtype, batch, pixels, channels, groups, null, null, pdtype, 1e-5, act, y, p256,
                                             ws, nbytes, null)

    def bwd(x=p256, dtype=0, batch=2, pixels=64, channels=32, groups=4, pdtype=0, act=1, dy=p256, ws=p256, nbytes=1 << 20):
        return lib.od_group_norm_act_backward(x, dy, dtype, batch, pixels, channels, groups, null, null, pdtype, act, p256, p256,
                                              null, null, ws, nbytes, null)
    for call in (fwd, bwd):
        assert call(x=null) == -1 and call(ws=null) == -1 and call(ws=p16) == -1
        assert call(dtype=3) == -1 and call(pdtype=-1) == -1 and call(act=3) == -1
        assert call(groups=0) == -1 and call(groups=5) == -1 and call(channels=0) == -1
        assert call(batch=-1) == -1 and call(pixels=-1) == -1
        assert call(channels=4096) == -2 and call(batch=65536) == -2
        assert call(nbytes=64) == -3
        assert call(x=ctypes.c_void_p(258)) == -1                                # not aligned to an element
        assert call(batch=0) == 0 and call(pixels=0) == 0
    assert fwd(y=null) == -1 and bwd(dy=null) == -1


def test_argument_errors_of_vocab_loss():
    lib = _C.lib()
    null, p16, p256 = ctypes.c_void_p(0), ctypes.c_void_p(16), ctypes.c_void_p(256)
    assert lib.od_vocab_loss_saved_bytes(1000, 1204, 256, 0, 2) >= 1024 * 256 * 2
    assert lib.od_vocab_loss_workspace_bytes(32768, 65536, 512, 0, 2, 1) < 32768 * 65536     # never the logits
    assert lib.od_vocab_loss_workspace_bytes(1000, 1204, 256, 8, 2, 0) > 0
    assert lib.od_vocab_loss_saved_bytes(10, 0, 256, 0, 2) == 0 and lib.od_vocab_loss_saved_bytes(10, 5, 0, 0, 2) == 0
    assert lib.od_vocab_loss_saved_bytes(10, 5, 8, 257, 2) == 0 and lib.od_vocab_loss_saved_bytes(10, 5, 16385, 0, 2) == 0
    assert lib.od_vocab_loss_saved_bytes(1 << 23, 5, 16384, 0, 0) == 0                       # 512 GiB of features
    assert lib.od_vocab_loss_saved_bytes((1 << 23) + 1, 5, 8, 0, 0) == 0

    def fwd(f=p256, fp=64, w=p256, wp=64, bias=null, dtype=2, rows=10, classes=50, dim=64, t=p256, top=0, tl=null, td=2, temp=1.0,
            red=1, loss=p256, saved=p256, ws=p256, nbytes=1 << 30):
        return lib.od_vocab_loss_forward(f, fp, w, wp, bias, dtype, rows, classes, dim, t, top, tl, td, temp, red, p256, loss,
                                         saved, nbytes, ws, nbytes, null)

    def bwd(w=p256, wp=64, bias=null, dtype=2, rows=10, classes=50, dim=64, t=p256, top=0, temp=1.0, red=1, up=p256, saved=p256,
            ws=p256, nbytes=1 << 30):
        return lib.od_vocab_loss_backward(w, wp, bias, dtype, rows, classes, dim, t, top, temp, red, up, saved, nbytes, p256,
                                          p256, null, ws, nbytes, null)
    for call in (fwd, bwd):
        assert call(w=null) == -1 and call(t=null) == -1 and call(saved=null) == -1 and call(ws=p16) == -1
        assert call(dtype=3) == -1 and call(red=3) == -1 and call(rows=-1) == -1 and call(classes=0) == -1 and call(dim=0) == -1
        assert call(top=-1) == -1 and call(temp=2.0) == -1                        # cross entropy has no temperature
        assert call(wp=63) == -1 and call(w=ctypes.c_void_p(257)) == -1
        assert call(top=257, temp=2.0) == -2 and call(dim=16385, wp=16385) == -2
        assert call(nbytes=1024) == -3
    assert fwd(f=null) == -1 and fwd(fp=63) == -1 and fwd(loss=null) == -1 and fwd(top=4) == -1     # no teacher logits
    assert fwd(top=4, tl=p256, temp=0.0) == -1 and fwd(top=4, tl=p256, temp=float("nan")) == -1
    assert fwd(top=4, tl=p256, td=5) == -1
    assert bwd(up=null) == -1 and bwd(rows=0) == 0


def test_temperatures_whose_square_leaves_fp32_are_refused():
    from object_detection_amd import det_utils
    lib = _C.lib()
    null, p256 = ctypes.c_void_p(0), ctypes.c_void_p(256)

    def fwd(temp, nbytes):
        return lib.od_vocab_loss_forward(p256, 64, p256, 64, null, 2, 10, 50, 64, p256, 4, p256, 2, temp, 1, p256, p256, p256,
                                         nbytes, p256, nbytes, null)
    for temp in (2.0 ** -64, 2.0 ** 64, 1e30, 1e-39, float("inf")):
        assert fwd(temp, 1024) == -1, temp
    for temp in (2.0 ** -63, 1.0, 2.0 ** 63):
        assert fwd(temp, 1024) == -3, temp                                      # stops at the workspace's size only
    features, weight = torch.zeros((2, 8)), torch.zeros((5, 8))
    logits, classes = torch.zeros((2, 3)), torch.zeros((2, 3), dtype=torch.int64)
    for temp in (0.0, -1.0, 1e30, 1e-30, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            det_utils.vocabulary_distillation(features, weight, logits, classes, temperature=temp)
