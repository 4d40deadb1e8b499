"""ctypes binding of libaiptd.so (include/aiptd.h) and a thin host-side mirror of the
reference's interface for the hot path.

Reference interface mirrored (Inference/src):
    pathtraceInit(Scene*) / pathtrace(pbo, frame, iter) / pathtraceFree()   pathtrace.h:6-8
    torch::jit::load + module.forward                                        main.cpp:104-111
    runCuda() per-frame body                                                 main.cpp:143-163

torch is used only as plumbing (device buffers, stream handles); every computation happens in
the HIP library.  There is no fallback: if libaiptd.so is missing or no GPU is visible, the
calls raise.
"""
from __future__ import annotations

import ctypes as C
import os
import struct

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("AIPT_LIB") or os.path.join(_HERE, "libaiptd.so")   # AIPT_LIB: kernel-variant builds (tools/)

# flags (include/aiptd.h)
TRACE_AA, TRACE_COMPACT, TRACE_RECORD_MAT0, TRACE_BRUTE_FORCE, TRACE_NO_BROAD_PHASE = 1, 2, 4, 8, 16
TRACE_SORT_MATERIAL, TRACE_CACHE_FIRST_BOUNCE, TRACE_MOTION_BLUR = 32, 64, 128
TRACE_NO_CULL, TRACE_DIELECTRIC, TRACE_MESH_NORMAL_VIEW = 512, 1024, 2048
SCENE_RECOMPUTE_NORMALS = 1
TRACE_DEFAULT = TRACE_AA | TRACE_COMPACT
DN_BN_BATCH, DN_BN_RUNNING, DN_HIDDEN_CARRY, DN_HIDDEN_RESET = 1, 0, 2, 0
DN_IMPL_MFMA, DN_IMPL_VALU, DN_IMPL_MFMA_F16X3, DN_IMPL_MFMA_F16W = 0, 1, 2, 3
DN_OPT_R_MINPIX, DN_OPT_F16_MINPIX, DN_OPT_SMALL_MINPIX, DN_OPT_FUSED_POOL, DN_OPT_KY_SPLIT = 1, 2, 3, 4, 5
GEOM_SPHERE, GEOM_CUBE = 0, 1
STREAM_DEFAULT = -1                                     # Context(stream=...): HIP's default stream, torch's own unless told otherwise
TYPE_F32, TYPE_BF16, TYPE_F16 = 0, 1, 2
ACTIVATIONS = {"none": 0, "leaky": 1, "silu": 2, "gelu": 3}
NORMS = {"rms": 0, "layer": 1}


class Geom(C.Structure):
    _fields_ = [("type", C.c_int), ("materialid", C.c_int),
                ("translation", C.c_float * 3), ("rotation", C.c_float * 3), ("scale", C.c_float * 3),
                ("transform", C.c_float * 16), ("inverseTransform", C.c_float * 16),
                ("invTranspose", C.c_float * 16), ("vel", C.c_float * 3)]


class Face(C.Structure):
    _fields_ = [("v", (C.c_float * 3) * 3), ("n", (C.c_float * 3) * 3), ("materialid", C.c_int)]


class Material(C.Structure):
    _fields_ = [("color", C.c_float * 3), ("specular_exponent", C.c_float), ("specular_color", C.c_float * 3),
                ("hasReflective", C.c_float), ("hasRefractive", C.c_float),
                ("indexOfRefraction", C.c_float), ("emittance", C.c_float)]


class Camera(C.Structure):
    _fields_ = [("resolution", C.c_int * 2), ("position", C.c_float * 3), ("lookAt", C.c_float * 3),
                ("view", C.c_float * 3), ("up", C.c_float * 3), ("right", C.c_float * 3),
                ("fov", C.c_float * 2), ("pixelLength", C.c_float * 2)]


class AABB(C.Structure):
    _fields_ = [("lb", C.c_float * 3), ("ub", C.c_float * 3)]


assert (C.sizeof(Geom), C.sizeof(Face), C.sizeof(Material), C.sizeof(Camera), C.sizeof(AABB)) == (248, 76, 44, 84, 24)


class LinearPlan(C.Structure):
    """aipt_linear_plan: which kernel a product is computed by"""
    _fields_ = [(n, C.c_int) for n in ("tile_rows", "tile_columns", "load", "lines", "copied", "splits")]


# every symbol include/aiptd.h declares: (name, restype, argtypes)
_P = C.c_void_p
ABI = [
    ("aipt_create", C.c_int, [C.c_int, _P, C.POINTER(_P)]),
    ("aipt_destroy", None, [_P]),
    ("aipt_stream", C.c_int, [_P, C.POINTER(_P)]),
    ("aipt_last_error", C.c_char_p, [_P]),
    ("aipt_abi_version", C.c_int, []),
    ("aipt_sync", C.c_int, [_P]),
    ("aipt_malloc", C.c_int, [_P, C.c_size_t, C.POINTER(_P)]),
    ("aipt_free", C.c_int, [_P, _P]),
    ("aipt_upload", C.c_int, [_P, _P, _P, C.c_size_t]),
    ("aipt_download", C.c_int, [_P, _P, _P, C.c_size_t]),
    ("aipt_memset", C.c_int, [_P, _P, C.c_int, C.c_size_t]),
    ("aipt_timer_start", C.c_int, [_P]),
    ("aipt_timer_stop", C.c_int, [_P, C.POINTER(C.c_float)]),
    ("aipt_scene_upload", C.c_int, [_P, _P, C.c_int, _P, C.c_int, _P, C.c_int, _P]),
    ("aipt_scene_free", C.c_int, [_P]),
    ("aipt_scene_pack", C.c_int, [_P, C.c_int, _P, C.c_int, _P, C.c_int, _P, C.POINTER(_P), C.POINTER(C.c_size_t), C.c_char_p,
                                  C.c_size_t]),
    ("aipt_blob_free", None, [_P]),
    ("aipt_scene_upload_packed", C.c_int, [_P, _P, C.c_size_t]),
    ("aipt_trace_configure_batch", C.c_int, [_P, C.c_int, C.c_int, C.c_int]),
    ("aipt_trace_batch", C.c_int, [_P, _P, C.c_int, C.c_int, C.c_int, C.c_uint32, _P, C.c_int, C.c_int, C.c_size_t]),
    ("aipt_trace_live_counts_frame", C.c_int, [_P, C.c_int, _P, C.c_int]),
    ("aipt_frames_configure", C.c_int, [_P, C.c_int]),
    ("aipt_frames", C.c_int, [_P, _P, C.c_int, C.c_int, C.c_int, C.c_uint32, C.c_uint32, C.c_uint32, _P]),
    ("aipt_frames_prefetch", C.c_int, [_P, _P, C.c_int, C.c_int, C.c_int, C.c_uint32]),
    ("aipt_frames_gbuffer", C.c_int, [_P, C.c_int, C.POINTER(_P), C.POINTER(C.c_int), C.POINTER(C.c_int)]),
    ("aipt_trace_profile_begin", C.c_int, [_P, C.c_int, C.c_int]),
    ("aipt_trace_profile_end", C.c_int, [_P, _P, C.c_int, C.POINTER(C.c_int)]),
    ("aipt_trace_profile_calls", C.c_int, [_P, _P, _P, C.c_int, C.c_int, C.POINTER(C.c_int)]),
    ("aipt_trace_kernel_name", C.c_int, [_P, C.c_int, C.c_char_p, C.c_size_t]),
    ("aipt_trace_configure", C.c_int, [_P, C.c_int, C.c_int]),
    ("aipt_trace", C.c_int, [_P, _P, C.c_int, C.c_int, C.c_uint32, _P, C.c_int, C.c_int]),
    ("aipt_debug_trace_stats", C.c_int, [_P, _P, C.c_int]),
    ("aipt_trace_live_counts", C.c_int, [_P, _P, C.c_int]),
    ("aipt_trace_first_hit_materials", C.c_int, [_P, _P, C.c_int]),
    ("aipt_denoise_load_weights", C.c_int, [_P, _P, C.c_size_t]),
    ("aipt_denoise_configure", C.c_int, [_P, C.c_int, C.c_int]),
    ("aipt_denoise_set_impl", C.c_int, [_P, C.c_int]),
    ("aipt_denoise_set_option", C.c_int, [_P, C.c_int, C.c_longlong]),
    ("aipt_denoise", C.c_int, [_P, _P, _P, C.c_uint32]),
    ("aipt_denoise_reset_hidden", C.c_int, [_P]),
    ("aipt_denoise_get_hidden", C.c_int, [_P, C.c_int, _P]),
    ("aipt_denoise_set_hidden", C.c_int, [_P, C.c_int, _P]),
    ("aipt_denoise_profile_begin", C.c_int, [_P, C.c_uint32, C.c_int]),
    ("aipt_denoise_profile_stride", C.c_int, [_P, C.c_int]),
    ("aipt_denoise_profile_end", C.c_int, [_P, _P, C.POINTER(C.c_int)]),
    ("aipt_denoise_layer_info", C.c_int, [_P, C.c_int, C.c_char_p, C.c_size_t] + [C.POINTER(C.c_int)] * 4
     + [C.POINTER(C.c_double)]),
    ("aipt_frame_configure", C.c_int, [_P, C.c_int, C.c_int]),
    ("aipt_frame", C.c_int, [_P, _P, C.c_int, C.c_int, C.c_uint32, C.c_uint32, _P]),
    ("aipt_gbuffer", C.c_int, [_P, C.POINTER(_P), C.POINTER(C.c_int), C.POINTER(C.c_int)]),
    ("aipt_frame_set_timing", C.c_int, [_P, C.c_int]),
    ("aipt_frame_last_times", C.c_int, [_P, C.POINTER(C.c_float), C.POINTER(C.c_float)]),
    ("aipt_frame_prefetch", C.c_int, [_P, _P, C.c_int, C.c_int, C.c_uint32]),
    ("aipt_linear_workspace", C.c_int, [_P, C.c_char_p, C.POINTER(C.c_size_t)]),
    ("aipt_linear", C.c_int, [_P, C.c_char_p, _P, C.c_size_t]),
    ("aipt_linear_planned", C.c_int, [_P, C.c_char_p, C.POINTER(LinearPlan)]),
    ("aipt_linear_backward_workspace", C.c_int, [_P, C.c_char_p, C.POINTER(C.c_size_t)]),
    ("aipt_linear_backward", C.c_int, [_P, C.c_char_p, _P, C.c_size_t]),
    ("aipt_linear_backward_planned", C.c_int, [_P, C.c_char_p, C.POINTER(LinearPlan), C.POINTER(LinearPlan)]),
    ("aipt_block_norm", C.c_int, [_P, C.c_char_p]),
    ("aipt_block_norm_backward_workspace", C.c_int, [_P, C.c_char_p, C.POINTER(C.c_size_t)]),
    ("aipt_block_norm_backward", C.c_int, [_P, C.c_char_p, _P, C.c_size_t]),
    ("aipt_adamw_state_elements", C.c_longlong, [_P, C.c_int]),
    ("aipt_adamw_workspace", C.c_longlong, [_P, C.c_int]),
    ("aipt_adamw_create", C.c_int, [_P, _P, C.c_int, C.c_int, C.c_int, C.c_int, _P, _P, _P, _P, _P, _P, _P, C.c_size_t, C.POINTER(_P)]),
    ("aipt_adamw_step", C.c_int, [_P, _P] + [C.c_double] * 5 + [C.c_uint32]),
    ("aipt_adamw_destroy", None, [_P]),
    ("aipt_comm_create", C.c_int, [C.POINTER(_P), C.c_int, C.c_int, C.POINTER(_P)]),
    ("aipt_comm_is_rccl", C.c_int, [_P]),
    ("aipt_comm_broadcast", C.c_int, [_P, C.POINTER(_P), C.c_size_t, C.c_int]),
    ("aipt_comm_destroy", None, [_P]),
    ("aipt_device_count", C.c_int, []),
    ("aipt_scene_load", C.c_int, [C.c_char_p, C.POINTER(_P), C.c_char_p, C.c_size_t]),
    ("aipt_scene_load_ex", C.c_int, [C.c_char_p, C.c_uint, C.POINTER(_P), C.c_char_p, C.c_size_t]),
    ("aipt_scene_release", None, [_P]),
    ("aipt_scene_set_resolution", C.c_int, [_P, C.c_int, C.c_int]),
    ("aipt_scene_info", C.c_int, [_P] + [C.POINTER(C.c_int)] * 5),
    ("aipt_scene_geoms", C.POINTER(Geom), [_P]),
    ("aipt_scene_materials", C.POINTER(Material), [_P]),
    ("aipt_scene_faces", C.POINTER(Face), [_P]),
    ("aipt_scene_mesh_box", C.POINTER(AABB), [_P]),
    ("aipt_scene_camera", C.c_int, [_P, C.POINTER(Camera)]),
    ("aipt_scene_orbit_params", C.c_int, [_P] + [C.POINTER(C.c_float)] * 3),
    ("aipt_scene_upload_host", C.c_int, [_P, _P]),
    ("aipt_geom_build", None, [C.POINTER(Geom)]),
    ("aipt_camera_orbit_params", None, [C.POINTER(Camera)] + [C.POINTER(C.c_float)] * 3),
    ("aipt_camera_orbit", None, [C.POINTER(Camera), C.c_float, C.c_float, C.c_float]),
]

# the argument records of the layer operators (include/aiptd.h), packed by field: a ctypes structure costs a small call more than its kernel
_LINEAR = struct.Struct("@iifi3q" + "Pqq" * 5 + "P")                 # aipt_linear_args
_LINEAR_GRAD = struct.Struct("@iifi3q" + "Pqq" * 6 + "P")            # aipt_linear_grad_args
_NORM = struct.Struct("@iifi2q4P4q6PP")                              # aipt_block_norm_args
_NORM_GRAD = struct.Struct("@4i2q4PP5P2P6q6P")                       # aipt_block_norm_grad_args
_ADAMW_TENSOR = struct.Struct("@3Pqfi")                              # aipt_adamw_tensor

_LIB = None


class AiptError(RuntimeError):
    pass


def lib():
    """Load libaiptd.so; raises if it has not been built (no fallback path exists)."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise AiptError(f"{LIB_PATH} not built: run `python -c 'import __graft_entry__ as g; g.build()'` "
                            "(hipcc --offload-arch=gfx950); this package has no CPU or PyTorch fallback")
        # torch bundles its own HIP runtime (torch/lib/libamdhip64.so, soname libamdhip64.so.7).  Import it first so
        # that libaiptd.so's DT_NEEDED libamdhip64.so.7 resolves to that already-loaded copy: two HIP runtimes in one
        # process leave the second one without a GPU ("No HIP GPUs are available").
        import torch  # noqa: F401
        L = C.CDLL(LIB_PATH)
        for name, res, args in ABI:
            fn = getattr(L, name)          # AttributeError if a declared symbol is not exported
            fn.restype = res
            fn.argtypes = args
        _LIB = L
    return _LIB


def scene_pack(geoms, materials, faces=(), mesh_box=None) -> bytes:
    """aipt_scene_pack: validate, build the mesh BVH once (host only) and return the relocatable scene blob that
    Context.pathtrace_init_packed uploads -- the unit rank 0 broadcasts to the other GPUs."""
    L = lib()
    ga = (Geom * max(1, len(geoms)))(*geoms)
    ma = (Material * max(1, len(materials)))(*materials)
    if isinstance(faces, np.ndarray):
        assert faces.dtype.itemsize == 76
        keep = np.ascontiguousarray(faces)
        fa = keep.ctypes.data_as(_P)
    else:
        fa = (Face * max(1, len(faces)))(*faces)
    box = mesh_box if mesh_box is not None else AABB()
    out, n = _P(), C.c_size_t()
    err = C.create_string_buffer(256)
    rc = L.aipt_scene_pack(ga, len(geoms), ma, len(materials), fa if len(faces) else None, len(faces),
                           C.byref(box) if len(faces) else None, C.byref(out), C.byref(n), err, 256)
    if rc:
        raise AiptError(f"aipt_scene_pack failed ({rc}): {err.value.decode()}")
    try:
        return C.string_at(out.value, n.value)
    finally:
        L.aipt_blob_free(out)


class Scene:
    """Host-side scene (reference class Scene, scene.h:13-44): parsed by the C++ front end of libaiptd.so."""

    def __init__(self, path: str, res=None, depth=None, flags=0):
        L = lib()
        h = _P()
        err = C.create_string_buffer(512)
        rc = L.aipt_scene_load_ex(path.encode(), int(flags), C.byref(h), err, 512)   # flags: SCENE_RECOMPUTE_NORMALS
        if rc:
            raise AiptError(f"aipt_scene_load({path}) failed ({rc}): {err.value.decode()}")
        self._h = h
        if res is not None:
            rc = L.aipt_scene_set_resolution(h, int(res[0]), int(res[1]))
            if rc:
                raise AiptError(f"aipt_scene_set_resolution{tuple(res)} failed ({rc})")
        n = [C.c_int() for _ in range(5)]
        L.aipt_scene_info(h, *[C.byref(v) for v in n])
        self.ngeoms, self.nmaterials, self.nfaces, self.iterations, self.depth = [v.value for v in n]
        if depth is not None:
            self.depth = depth
        self.camera = Camera()
        L.aipt_scene_camera(h, C.byref(self.camera))
        z, p, t = C.c_float(), C.c_float(), C.c_float()
        L.aipt_scene_orbit_params(h, C.byref(z), C.byref(p), C.byref(t))
        self.zoom, self.phi, self.theta = z.value, p.value, t.value

    def close(self):
        if getattr(self, "_h", None):
            lib().aipt_scene_release(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def geoms(self):
        p = lib().aipt_scene_geoms(self._h)
        return [p[i] for i in range(self.ngeoms)]

    @property
    def materials(self):
        p = lib().aipt_scene_materials(self._h)
        return [p[i] for i in range(self.nmaterials)]

    @property
    def faces(self):
        p = lib().aipt_scene_faces(self._h)
        return [p[i] for i in range(self.nfaces)]

    @property
    def mesh_box(self):
        return lib().aipt_scene_mesh_box(self._h).contents

    def orbit(self, zoom=None, phi=None, theta=None) -> Camera:
        """runCuda() camera rebuild (main.cpp:122-140); returns a Camera for this frame."""
        cam = Camera.from_buffer_copy(bytes(self.camera))
        lib().aipt_camera_orbit(C.byref(cam), self.zoom if zoom is None else zoom,
                                self.phi if phi is None else phi, self.theta if theta is None else theta)
        return cam


class Context:
    """One context per GPU (aipt_create).  stream: a raw hipStream_t handle (int), STREAM_DEFAULT (torch's default stream) or None (a stream of
    the context's own)."""

    def __init__(self, device: int = 0, stream=None):
        L = lib()
        h = _P()
        rc = L.aipt_create(device, _P(stream) if stream else None, C.byref(h))
        if rc:
            raise AiptError(f"aipt_create failed ({rc}): {L.aipt_last_error(None).decode()}")
        self._h = h
        self.device = device
        self._keep = []
        self._stream, self._ext = None, None             # of the layer operators: the context's stream (handle; torch object)

    def close(self):
        if getattr(self, "_h", None):
            lib().aipt_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _ck(self, rc):
        if rc:
            raise AiptError(f"libaiptd error {rc}: {lib().aipt_last_error(self._h).decode()}")

    def sync(self):
        self._ck(lib().aipt_sync(self._h))

    def timer_start(self):
        self._ck(lib().aipt_timer_start(self._h))

    def timer_stop(self) -> float:
        ms = C.c_float()
        self._ck(lib().aipt_timer_stop(self._h, C.byref(ms)))
        return ms.value

    # ------------------------------------------------------------------ trace (pathtrace.h:6-8)
    def pathtrace_init(self, geoms, materials, faces=(), mesh_box=None, width=None, height=None):
        """pathtraceInit(Scene*): upload the scene; allocate path state for width x height."""
        ga = (Geom * max(1, len(geoms)))(*geoms)
        ma = (Material * max(1, len(materials)))(*materials)
        if isinstance(faces, np.ndarray):                      # structured array with the 76-byte Face layout
            assert faces.dtype.itemsize == 76
            keep = np.ascontiguousarray(faces)
            fa = keep.ctypes.data_as(_P)
        else:
            fa = (Face * max(1, len(faces)))(*faces)
        box = mesh_box if mesh_box is not None else AABB()
        self._ck(lib().aipt_scene_upload(self._h, ga, len(geoms), ma, len(materials),
                                         fa if len(faces) else None, len(faces),
                                         C.byref(box) if len(faces) else None))
        if width is not None:
            self._ck(lib().aipt_trace_configure(self._h, width, height))

    def pathtrace_init_packed(self, blob: bytes, width=None, height=None):
        """pathtraceInit from a packed scene (scene_pack): copies only, the BVH inside the blob is not rebuilt."""
        self._ck(lib().aipt_scene_upload_packed(self._h, blob, len(blob)))
        if width is not None:
            self._ck(lib().aipt_trace_configure(self._h, width, height))

    def trace_profile_begin(self, max_calls: int, every: int = 1):
        self._ck(lib().aipt_trace_profile_begin(self._h, max_calls, every))

    def trace_profile_end(self, nbounces: int):
        """-> (summed ms of every bounce launch [nbounces], number of recorded traces)"""
        ms = np.zeros(nbounces, np.float64)
        n = C.c_int()
        self._ck(lib().aipt_trace_profile_end(self._h, ms.ctypes.data, nbounces, C.byref(n)))
        return ms, n.value

    def trace_profile_calls(self, nbounces: int, max_calls: int = 4096):
        """-> (frames held by every recorded trace call [calls], ms of its bounce launches [calls, nbounces]); before _end"""
        fr = np.zeros(max_calls, np.int32)
        ms = np.zeros((max_calls, nbounces), np.float64)
        n = C.c_int()
        self._ck(lib().aipt_trace_profile_calls(self._h, fr.ctypes.data, ms.ctypes.data, nbounces, max_calls, C.byref(n)))
        return fr[:n.value].copy(), ms[:n.value].copy()

    def trace_kernel_name(self, bounce: int) -> str:
        name = C.create_string_buffer(64)
        self._ck(lib().aipt_trace_kernel_name(self._h, bounce, name, 64))
        return name.value.decode()

    def pathtrace_init_scene(self, scene: "Scene", width=None, height=None):
        """pathtraceInit(Scene*) from a parsed Scene."""
        self._ck(lib().aipt_scene_upload_host(self._h, scene._h))
        if width is not None:
            self._ck(lib().aipt_trace_configure(self._h, width, height))

    def pathtrace_free(self):
        self._ck(lib().aipt_scene_free(self._h))

    def pathtrace(self, cam: Camera, iter: int, depth: int, gbuf, flags: int = TRACE_DEFAULT):
        """pathtrace(pbo, frame, iter): one 1-spp iteration into gbuf, a float32 device tensor [10, rows, stride]."""
        assert gbuf.is_cuda and gbuf.dtype.is_floating_point and gbuf.dim() == 3 and gbuf.shape[0] == 10
        assert gbuf.is_contiguous()
        self._ck(lib().aipt_trace(self._h, C.byref(cam), iter, depth, flags, _P(gbuf.data_ptr()),
                                  gbuf.shape[1], gbuf.shape[2]))

    def live_counts(self, depth: int) -> np.ndarray:
        out = np.zeros(depth + 1, np.int32)
        self._ck(lib().aipt_trace_live_counts(self._h, out.ctypes.data, depth + 1))
        return out

    def first_hit_materials(self, n: int) -> np.ndarray:
        out = np.zeros(n, np.int32)
        self._ck(lib().aipt_trace_first_hit_materials(self._h, out.ctypes.data, n))
        return out

    # ------------------------------------------------------------------ denoiser (main.cpp:101-118)
    def load_weights(self, blob: bytes):
        """torch::jit::load(MODEL_PATH) counterpart: flat blob (arch.py)."""
        self._ck(lib().aipt_denoise_load_weights(self._h, blob, len(blob)))

    def denoise_configure(self, H: int, W: int):
        self._ck(lib().aipt_denoise_configure(self._h, H, W))

    def denoise_set_impl(self, impl: int):
        self._ck(lib().aipt_denoise_set_impl(self._h, impl))

    def denoise_set_option(self, option, value):
        """aipt_denoise_set_option: DN_OPT_R_MINPIX / DN_OPT_F16_MINPIX / DN_OPT_SMALL_MINPIX / DN_OPT_FUSED_POOL / DN_OPT_KY_SPLIT"""
        self._ck(lib().aipt_denoise_set_option(self._h, option, value))

    def denoise(self, x10, out3, bn_batch: bool = True, carry: bool = False):
        """module.forward: x10 [10,H,W] -> out3 [3,H,W], float32 contiguous device tensors."""
        assert x10.is_cuda and out3.is_cuda and x10.is_contiguous() and out3.is_contiguous()
        flags = (DN_BN_BATCH if bn_batch else 0) | (DN_HIDDEN_CARRY if carry else 0)
        self._ck(lib().aipt_denoise(self._h, _P(x10.data_ptr()), _P(out3.data_ptr()), flags))

    def reset_hidden(self):
        self._ck(lib().aipt_denoise_reset_hidden(self._h))

    def get_hidden(self, level: int, dst):
        self._ck(lib().aipt_denoise_get_hidden(self._h, level, _P(dst.data_ptr())))

    def set_hidden(self, level: int, src):
        self._ck(lib().aipt_denoise_set_hidden(self._h, level, _P(src.data_ptr())))

    def profile_begin(self, layer_mask: int, max_calls: int):
        self._ck(lib().aipt_denoise_profile_begin(self._h, layer_mask, max_calls))

    def profile_end(self):
        """-> (summed ms per layer [28], number of recorded forwards)"""
        ms = np.zeros(28, np.float64)
        n = C.c_int()
        self._ck(lib().aipt_denoise_profile_end(self._h, ms.ctypes.data, C.byref(n)))
        return ms, n.value

    def profile_stride(self, every: int):
        self._ck(lib().aipt_denoise_profile_stride(self._h, every))

    def layer_info(self, layer: int):
        name = C.create_string_buffer(64)
        ci, co, h, w = C.c_int(), C.c_int(), C.c_int(), C.c_int()
        fl = C.c_double()
        self._ck(lib().aipt_denoise_layer_info(self._h, layer, name, 64, C.byref(ci), C.byref(co), C.byref(h),
                                               C.byref(w), C.byref(fl)))
        return dict(kernel=name.value.decode(), cin=ci.value, cout=co.value, h=h.value, w=w.value, flops=fl.value)

    # ------------------------------------------------------------------ frame (runCuda, main.cpp:143-163)
    def frame_configure(self, width: int, height: int):
        self._ck(lib().aipt_frame_configure(self._h, width, height))

    def frame(self, cam: Camera, iter: int, depth: int, out3, trace_flags: int = TRACE_DEFAULT,
              bn_batch: bool = True, carry: bool = True):
        flags = (DN_BN_BATCH if bn_batch else 0) | (DN_HIDDEN_CARRY if carry else 0)
        self._ck(lib().aipt_frame(self._h, C.byref(cam), iter, depth, trace_flags, flags, _P(out3.data_ptr())))

    def trace_configure_batch(self, width: int, height: int, batch: int):
        self._ck(lib().aipt_trace_configure_batch(self._h, width, height, batch))

    def pathtrace_batch(self, cams, iter: int, depth: int, gbufs, flags: int = TRACE_DEFAULT):
        """aipt_trace_batch: len(cams) frames into gbufs, a float32 device tensor [nframes, 10, rows, stride]"""
        assert gbufs.is_cuda and gbufs.is_contiguous() and gbufs.dim() == 4 and gbufs.shape[0] >= len(cams) and gbufs.shape[1] == 10
        ca = (Camera * len(cams))(*cams)
        self._ck(lib().aipt_trace_batch(self._h, ca, len(cams), iter, depth, flags, _P(gbufs.data_ptr()), gbufs.shape[2],
                                        gbufs.shape[3], 10 * gbufs.shape[2] * gbufs.shape[3]))

    def live_counts_frame(self, frame: int, depth: int) -> np.ndarray:
        out = np.zeros(depth + 1, np.int32)
        self._ck(lib().aipt_trace_live_counts_frame(self._h, frame, out.ctypes.data, depth + 1))
        return out

    def frames_configure(self, batch: int):
        self._ck(lib().aipt_frames_configure(self._h, batch))

    def frames(self, cams, iter: int, depth: int, outs, trace_flags: int = TRACE_DEFAULT, bn_batch: bool = True,
               carry_first: bool = True, carry: bool = True):
        """aipt_frames: trace len(cams) consecutive frames with one set of launches, denoise them in order into outs[j]."""
        ca = (Camera * len(cams))(*cams)
        ptrs = (_P * len(cams))(*[_P(o.data_ptr()) for o in outs[:len(cams)]])
        f0 = (DN_BN_BATCH if bn_batch else 0) | (DN_HIDDEN_CARRY if carry_first else 0)
        f1 = (DN_BN_BATCH if bn_batch else 0) | (DN_HIDDEN_CARRY if carry else 0)
        self._ck(lib().aipt_frames(self._h, ca, len(cams), iter, depth, trace_flags, f0, f1, ptrs))

    def frames_prefetch(self, cams, iter: int, depth: int, trace_flags: int = TRACE_DEFAULT):
        ca = (Camera * len(cams))(*cams)
        self._ck(lib().aipt_frames_prefetch(self._h, ca, len(cams), iter, depth, trace_flags))

    def frames_gbuffer(self, frame: int):
        p, r, s = _P(), C.c_int(), C.c_int()
        self._ck(lib().aipt_frames_gbuffer(self._h, frame, C.byref(p), C.byref(r), C.byref(s)))
        return p.value, r.value, s.value

    def frame_prefetch(self, cam: Camera, iter: int, depth: int, trace_flags: int = TRACE_DEFAULT):
        """Trace the NEXT frame on the side stream while the current one is denoised; the next frame() call with the
        same arguments consumes it."""
        self._ck(lib().aipt_frame_prefetch(self._h, C.byref(cam), iter, depth, trace_flags))

    def gbuffer(self):
        """(device pointer, rows, stride) of the context-owned padded G-buffer."""
        p, r, s = _P(), C.c_int(), C.c_int()
        self._ck(lib().aipt_gbuffer(self._h, C.byref(p), C.byref(r), C.byref(s)))
        return p.value, r.value, s.value

    def frame_set_timing(self, on: bool):
        self._ck(lib().aipt_frame_set_timing(self._h, 1 if on else 0))

    def frame_last_times(self):
        a, b = C.c_float(), C.c_float()
        self._ck(lib().aipt_frame_last_times(self._h, C.byref(a), C.byref(b)))
        return a.value, b.value

    # ------------------------------------------------------------------ layer operators
    # Tensors are torch's; the work runs on the context's stream.  Where that is not torch's current stream, the call waits for what is
    # queued there and what is queued there later waits for the call, so that tensors may be used, and freed, like in any torch program.  Autograd
    # records none of these calls (gradients are the _backward methods'), but it is told what they write: a tensor that it saved for a backward pass
    # of its own and that is written since is refused there.
    def _on_stream(self, entry, *args):
        if not self._h:
            raise AiptError("the context is closed")
        if self._stream is None:
            import torch
            p = _P()
            self._ck(lib().aipt_stream(self._h, C.byref(p)))
            self._stream = p.value or 0
            # (ExternalStream takes 0 for "none given" and makes a new stream)
            self._ext = torch.cuda.ExternalStream(self._stream, device=self.device) if self._stream else torch.cuda.default_stream(self.device)
            self._current = torch._C._cuda_getCurrentRawStream
        if self._current(self.device) == self._stream:
            rc = entry(self._h, *args)
            return self._ck(rc) if rc else None
        import torch
        now = torch.cuda.current_stream(self.device)
        if not self._stream and self._capturing():
            raise AiptError("a context on the default stream cannot take part in a capture: make one with stream=<the capturing stream's handle>")
        self._ext.wait_stream(now)
        rc = entry(self._h, *args)
        now.wait_stream(self._ext)
        self._ck(rc)

    def _capturing(self, stream=None) -> bool:
        """Is this stream, or torch's current one of this device, being captured?"""
        import torch
        if stream is not None:
            with torch.cuda.stream(stream):
                return torch._C._cuda_isCurrentStreamCapturing()
        if torch._C._cuda_getDevice() == self.device:
            return torch._C._cuda_isCurrentStreamCapturing()
        with torch.cuda.device(self.device):
            return torch._C._cuda_isCurrentStreamCapturing()

    def _scratch(self, entry, record):
        """(memory or None, its address, bytes) of an operator's workspace: torch's, so that a captured graph keeps its own"""
        n = C.c_size_t()
        self._ck(entry(self._h, record, C.byref(n)))
        size = n.value
        if not size:
            return None, None, 0
        import torch
        t = torch.empty(size, dtype=torch.uint8, device=self.device)
        return t, t.data_ptr(), size

    def _type(self, t):
        kind = _types().get(t.dtype)
        if kind is None or t.get_device() != self.device:
            raise AiptError(f"a {t.dtype} tensor on {t.device}: float32, bfloat16 or float16 on cuda:{self.device} is wanted")
        return kind

    # (get_device() is -1 of a CPU tensor; a shape compares like a tuple)
    def _want(self, name, t, dtype, *shape):
        if t.dtype is not dtype or t.get_device() != self.device or t.shape != shape:
            raise AiptError(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}; {dtype} {shape} on cuda:{self.device} is wanted")

    def _matrix(self, name, t, dtype, rows, cols):
        """(address, row stride, column stride) of an optional matrix"""
        if t is None:
            return 0, 0, 0
        if t.dtype is not dtype or t.get_device() != self.device or t.shape != (rows, cols):
            self._want(name, t, dtype, rows, cols)
        return (t.data_ptr(), *t.stride())

    def _vector(self, name, t, dtype, n):
        if t is None:
            return 0
        if t.dtype is not dtype or t.get_device() != self.device or t.shape != (n,):
            self._want(name, t, dtype, n)
        if n > 1 and t.stride(0) != 1:
            raise AiptError(f"{name}: stride {t.stride(0)}")
        return t.data_ptr()

    # the same of several at once: a call of little work is bound by what is done here for each tensor
    def _vectors(self, dtype, n, **of):
        dev, shape = self.device, (n,)
        return [0 if t is None else t.data_ptr() if t.dtype is dtype and t.get_device() == dev and t.shape == shape and t.is_contiguous()
                else self._vector(name, t, dtype, n) for name, t in of.items()]

    def linear(self, x, w, y, bias=None, residual=None, preact=None, act: str = "none", slope: float = 0.1):
        """aipt_linear: y = act(x w^T + bias) + residual.  x [m, k], w [n, k], y [m, n] -- each with unit stride along either axis, so a planar
        feature map [channels, pixels] comes as its .t() -- bias [n], residual [m, n] (may be y); preact [m, n] receives x w^T + bias, which
        linear_backward of an activation wants.  All float32, bfloat16 or float16.  act: none, leaky (slope), silu, gelu."""
        kind, d = self._type(x), x.dtype
        if x.dim() != 2 or w.dim() != 2:
            raise AiptError(f"linear: x {tuple(x.shape)}, w {tuple(w.shape)}")
        (m, k), n = x.shape, w.shape[0]
        record = _LINEAR.pack(kind, _choice("act", act, ACTIVATIONS), slope, 0, m, n, k, *self._matrix("x", x, d, m, k), *self._matrix("w", w, d, n, k),
                              *self._matrix("y", y, d, m, n), *self._matrix("residual", residual, d, m, n),
                              *self._matrix("preact", preact, d, m, n), self._vector("bias", bias, d, n))
        hold, ptr, size = self._scratch(lib().aipt_linear_workspace, record)
        self._on_stream(lib().aipt_linear, record, ptr, size)
        _written(y, preact)
        return y

    def linear_backward(self, dy, x, w, preact=None, act: str = "none", slope: float = 0.1, dx=None, dw=None, dbias=None):
        """aipt_linear_backward: gradients of linear() into dx [m, k], dw [n, k], dbias [n], each or None (the residual's is dy).  preact: what
        linear() kept; not needed with act "none".  x is looked at for dw alone, w for dx alone: either may be None without."""
        kind, d = self._type(dy), dy.dtype
        if dy.dim() != 2:
            raise AiptError(f"linear_backward: dy {tuple(dy.shape)}")
        if (dw is not None and x is None) or (dx is not None and w is None):
            raise AiptError("linear_backward: dw wants x, dx wants w")
        (m, n), like = dy.shape, x if x is not None else w if w is not None else None
        if like is not None and like.dim() != 2:
            raise AiptError(f"linear_backward: x or w {tuple(like.shape)}")
        k = like.shape[1] if like is not None else 0
        act = _choice("act", act, ACTIVATIONS)
        if act and preact is None:
            raise AiptError("linear_backward: an activation wants preact")
        record = _LINEAR_GRAD.pack(kind, act, slope, 0, m, n, k, *self._matrix("dy", dy, d, m, n), *self._matrix("x", x, d, m, k),
                                   *self._matrix("w", w, d, n, k), *self._matrix("preact", preact, d, m, n), *self._matrix("dx", dx, d, m, k),
                                   *self._matrix("dw", dw, d, n, k), self._vector("dbias", dbias, d, n))
        hold, ptr, size = self._scratch(lib().aipt_linear_backward_workspace, record)
        self._on_stream(lib().aipt_linear_backward, record, ptr, size)
        _written(dx, dw, dbias)

    def _rows(self, dtype, rows, c, **of):
        """the addresses and the row strides of optional [rows, c] with contiguous rows"""
        dev, shape, at, strides = self.device, (rows, c), [], []
        for name, t in of.items():
            if t is None:
                at.append(0)
                strides.append(0)
                continue
            if t.dtype is not dtype or t.get_device() != dev or t.shape != shape:
                self._want(name, t, dtype, rows, c)
            row, col = t.stride()
            if col != 1 and c > 1:
                raise AiptError(f"{name}: stride {col} between the channels of a row")
            at.append(t.data_ptr())
            strides.append(row)
        return at, strides

    def _gates(self, name, t, dtype, c, groups):
        if t is None:
            return 0
        if t.dtype is not dtype or t.get_device() != self.device or t.shape != (groups, c) or not t.is_contiguous():
            if t.dim() != 2 or not t.is_contiguous():
                raise AiptError(f"{name}: {tuple(t.shape)} contiguous [groups, channels] is wanted")
            self._want(name, t, dtype, groups, c)
        return t.data_ptr()

    def _stats(self, stats, rows):
        if stats is None:
            return 0
        if _TYPES.get(stats.dtype) != TYPE_F32 or stats.get_device() != self.device or stats.shape != (rows, 4) or not stats.is_contiguous():
            import torch
            self._want("stats", stats, torch.float32, rows, 4)
            if not stats.is_contiguous():
                raise AiptError("stats is not contiguous")
        return stats.data_ptr()

    def block_norm(self, y, x, h, z=None, gate=None, scale=None, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None, kind: str = "rms",
                   eps: float = 1e-5, stats=None):
        """aipt_block_norm: the norm behind a residual block, its gate and residual scale, and the norm before the next block:
        h = x + scale * gate * (norm(y) * post_weight + post_bias), z = norm(h) * pre_weight + pre_bias.  y (None: no block yet, h = x), x, h (may
        be x), z (None: no norm) [rows, channels]; gate [groups, channels], one for each rows / groups rows; the rest [channels]; stats
        float32 [rows, 4] receives what block_norm_backward wants.  kind: rms, or layer (which alone has biases)."""
        t, d = self._type(x), x.dtype
        if x.dim() != 2:
            raise AiptError(f"block_norm: x {tuple(x.shape)}")
        rows, c = x.shape
        groups = gate.shape[0] if gate is not None and gate.dim() == 2 else 1
        at, strides = self._rows(d, rows, c, x=x, y=y, h=h, z=z)
        record = _NORM.pack(t, _choice("kind", kind, NORMS), eps, c, rows, groups, *at, *strides, self._gates("gate", gate, d, c, groups),
                            *self._vectors(d, c, scale=scale, post_weight=post_weight, post_bias=post_bias, pre_weight=pre_weight, pre_bias=pre_bias), self._stats(stats, rows))
        self._on_stream(lib().aipt_block_norm, record)
        _written(h, z, stats)
        return h, z

    def block_norm_backward(self, dh, dz, y, h, stats, gate=None, scale=None, post_weight=None, post_bias=None, pre_weight=None, kind: str = "rms",
                            dx=None, dy=None, dgate=None, dscale=None, dpost_weight=None, dpost_bias=None, dpre_weight=None, dpre_bias=None):
        """aipt_block_norm_backward: gradients of block_norm() from dh (None: zero) and dz (None: there was no z), with y, h and stats as it left
        them, into dx (may be dh), dy and the parameters' gradients, each or None."""
        like = dh if dh is not None else dz
        if like is None or like.dim() != 2:
            raise AiptError("block_norm_backward: dh or dz [rows, channels] is wanted")
        t, d = self._type(like), like.dtype
        rows, c = like.shape
        g = gate if gate is not None else dgate
        groups = g.shape[0] if g is not None and g.dim() == 2 else 1
        at, strides = self._rows(d, rows, c, dh=dh, dz=dz, y=y, h=h, dx=dx, dy=dy)
        vec = self._vectors(d, c, scale=scale, post_weight=post_weight, post_bias=post_bias, pre_weight=pre_weight, dscale=dscale, dpost_weight=dpost_weight,
                            dpost_bias=dpost_bias, dpre_weight=dpre_weight, dpre_bias=dpre_bias)
        record = _NORM_GRAD.pack(t, _choice("kind", kind, NORMS), c, 0, rows, groups, *at[:4], self._stats(stats, rows), self._gates("gate", gate, d, c, groups),
                                 *vec[:4], *at[4:], *strides, self._gates("dgate", dgate, d, c, groups), *vec[4:])
        hold, ptr, size = self._scratch(lib().aipt_block_norm_backward_workspace, record)
        self._on_stream(lib().aipt_block_norm_backward, record, ptr, size)
        _written(dx, dy, dgate, dscale, dpost_weight, dpost_bias, dpre_weight, dpre_bias)

    def adamw(self, params, grads, copies=None, weight_decay=0.01, state_bits: int = 32, state=None) -> "AdamW":
        """A plan for AdamW steps over these tensors (class AdamW)."""
        return AdamW(self, params, grads, copies, weight_decay, state_bits, state)


def _types():
    global _TYPES
    if _TYPES is None:
        import torch
        _TYPES = {torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16, torch.float16: TYPE_F16}
    return _TYPES


_TYPES = None
_INCREMENT = None


def _written(*tensors):
    """These were written through their addresses, which torch does not see: their versions go on, as after an operation in place."""
    global _INCREMENT
    if _INCREMENT is None:
        import torch
        _INCREMENT = torch.autograd.graph.increment_version
    _INCREMENT([t for t in tensors if t is not None])


def _choice(name, value, choices):
    if value not in choices:
        raise AiptError(f"{name} {value!r}: one of {', '.join(choices)} is wanted")
    return choices[value]


class AdamW:
    """AdamW over many tensors at once (aipt_adamw_*; the reference trains with torch's Adam, training/train.py:54-112).

    params: contiguous float32 tensors; grads: as many, of the same sizes, all float32, bfloat16 or float16; copies: None, or bfloat16 or
    float16 tensors that receive the rounded parameters (an entry may be None); weight_decay: a number, or one for each tensor.  The plan is
    bound to these tensors' memory: a gradient that is replaced by another tensor, or storage that moves, is bound anew with bind(); where a gradient is its
    parameter's .grad, update() refuses to step with one that is so no longer.
    state: None (zeros, step 0) or the dict that state() of an earlier plan of the same sizes returned, which goes on being updated in place:
    step int32 [1]; m and v float32 (state_bits 32), or m, v float8_e4m3fn with m_scale, v_scale float32 for each 256 elements (state_bits
    8; v holds the second moment's root); tensor i begins at element 256 * (number of 256-blocks of the tensors before it).
    norm: float32 [1], the gradients' norm at the last update that clipped.
    A graph that captured update() steps the tensors that were bound then, whatever is bound later, as long as this object lives."""

    def __init__(self, ctx, params, grads, copies=None, weight_decay=0.01, state_bits=32, state=None):
        import torch
        self.ctx, self._h = ctx, None
        params = list(params)
        copies = list(copies) if copies is not None else [None] * len(params)
        decay = [float(weight_decay)] * len(params) if isinstance(weight_decay, (int, float)) else [float(v) for v in weight_decay]
        if not (len(params) == len(copies) == len(decay)):
            raise AiptError(f"adamw: {len(params)} params, {len(copies)} copies, {len(decay)} weight_decay")
        if state_bits not in (8, 32):
            raise AiptError(f"adamw: state_bits {state_bits}: 32 or 8 is wanted")
        self._params, self._copies, self._decay, self.state_bits = params, copies, decay, state_bits
        dev = torch.device("cuda", ctx.device)
        n = len(params)
        counts = (C.c_longlong * max(1, n))(*[p.numel() for p in params])
        total, need = lib().aipt_adamw_state_elements(counts, n), lib().aipt_adamw_workspace(counts, n)
        if total < 0 or need < 0:
            raise AiptError("adamw: a tensor has too many elements")
        kind, blocks = torch.float32 if state_bits == 32 else torch.float8_e4m3fn, total // 256
        want = {"m": (kind, total), "v": (kind, total), "step": (torch.int32, 1)}
        if state_bits == 8:
            want.update(m_scale=(torch.float32, blocks), v_scale=(torch.float32, blocks))
        if state is None:
            state = {k: torch.zeros(size, device=dev, dtype=torch.uint8 if t.itemsize == 1 else t).view(t) for k, (t, size) in want.items()}
        if set(state) != set(want):
            raise AiptError(f"adamw: state has {sorted(state)}, {sorted(want)} are wanted")
        for k, (t, size) in want.items():
            ctx._want("state " + k, state[k], t, size)
            if not state[k].is_contiguous():
                raise AiptError(f"adamw: state {k} is not contiguous")
        self._state = dict(state)
        self.norm = torch.zeros(1, device=dev)
        self._need, self._captured, self._kept, self._homes = need, None, [], [None]
        self.bind(grads)

    def bind(self, grads):
        """Bind the plan to these gradients, and to where the parameters and copies lie now.  Waits for the stream; not in a capture."""
        import torch
        grads, ctx = list(grads), self.ctx
        if len(grads) != len(self._params):
            raise AiptError(f"adamw: {len(self._params)} params, {len(grads)} grads")
        kinds = {g.dtype for g in grads} or {torch.float32}
        copies = {c.dtype for c in self._copies if c is not None} or {torch.bfloat16}
        if len(kinds) != 1 or not kinds <= set(_types()) or len(copies) != 1 or not copies <= {torch.bfloat16, torch.float16}:
            raise AiptError("adamw: gradients of one type (float32, bfloat16, float16) and copies of one (bfloat16, float16) are wanted")
        records = []
        for i, (p, g, c, d) in enumerate(zip(self._params, grads, self._copies, self._decay)):
            for name, t, kind in (("param", p, torch.float32), ("grad", g, g.dtype), ("copy", c, None if c is None else c.dtype)):
                if t is not None:
                    ctx._want(f"{name} {i}", t, kind, *p.shape)
                    if not t.is_contiguous():
                        raise AiptError(f"adamw: {name} {i} is not contiguous")
            records.append(_ADAMW_TENSOR.pack(p.data_ptr(), g.data_ptr(), 0 if c is None else c.data_ptr(), p.numel(), d, 0))
        s, h = self._state, _P()
        ptr = {k: s[k].data_ptr() if k in s else None for k in ("m", "v", "m_scale", "v_scale", "step")}
        if ctx._capturing():
            raise AiptError("adamw: a plan is made, and bound, before a capture")
        # Each binding has a table of its own: a graph that captured a step reads that binding's, and steps of it may still run.
        # (in the streams' order: the table is written behind the zeros)
        scratch = torch.zeros(self._need, device=s["step"].device, dtype=torch.uint8)
        ctx._on_stream(lib().aipt_adamw_create, b"".join(records), len(records), _types()[kinds.pop()], _types()[copies.pop()], self.state_bits, ptr["m"], ptr["v"],
                       ptr["m_scale"], ptr["v_scale"], ptr["step"], self.norm.data_ptr(), scratch.data_ptr(), scratch.numel(), C.byref(h))
        if self._captured:
            self._kept.append(self._captured)
        self.close()
        self._h, self._grads, self._scratch, self._captured = h, grads, scratch, None
        home = None if ctx._ext is None else torch.cuda.current_stream(ctx.device)
        if home not in self._homes:
            self._homes.append(home)
        self._held = [t for t in (*self._params, *grads, *self._copies, *s.values()) if t is not None]
        bases = [t if t._base is None else t._base for t in (*self._params, *self._copies) if t is not None]      # views of one tensor count as it does
        self._steps_on = list({id(t): t for t in bases}.values())
        self._own_grads = [(p, g) for p, g in zip(self._params, grads) if p.is_leaf and p.grad is g]
        self._address = torch.Tensor.data_ptr
        self._at = list(map(self._address, self._held))

    def state(self) -> dict:
        """The state tensors themselves, to be saved, or to go on from in another plan."""
        return dict(self._state)

    def update(self, lr: float, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8, max_norm: float = None, seed: int = 0):
        """One step.  max_norm: clip the gradients' norm to this (None: no clipping); a step whose norm is not finite then changes nothing.  seed: key of
        the chances by which 8-bit state is rounded.  A captured step replays its lr; the step number goes on with every replay."""
        if not self._h:
            raise AiptError("adamw: the plan is closed")
        if list(map(self._address, self._held)) != self._at:
            raise AiptError("adamw: a tensor's storage has moved: bind() the plan anew")
        for p, g in self._own_grads:
            if p.grad is not g:
                raise AiptError("adamw: a parameter's .grad is none or another tensor than the plan was bound to: bind() the plan anew, or keep gradients (zero_grad(set_to_none=False))")
        if max_norm is not None and not max_norm > 0:
            raise AiptError(f"adamw: max_norm {max_norm}")
        if not self._captured and self.ctx._capturing():
            self._captured = [self._scratch, *(t.detach() for t in self._held)]      # the graph's: kept, wherever these tensors' storage moves
        self.ctx._on_stream(lib().aipt_adamw_step, self._h, lr, beta1, beta2, eps, 0.0 if max_norm is None else max_norm, seed & 0xffffffff)
        _written(*self._steps_on)

    def _release(self):
        """Memory of the plan may be freed next.  Every step runs on the context's stream, whatever stream it was queued from: the streams that the
        memory was taken on wait for it, so that who gets it there does not write under a step.  (A closed context's stream is done.)"""
        ctx = self.ctx
        if not ctx._h or ctx._ext is None:
            return
        homes = [s for s in self._homes if s is not None and s != ctx._ext]
        if homes and any(map(ctx._capturing, (ctx._ext, *homes))):
            ctx._keep.append((self._scratch, self.norm, self._state))         # no waiting into a capture or out of one
            return
        for s in homes:
            s.wait_stream(ctx._ext)

    def close(self):
        if getattr(self, "_h", None):
            self._release()
            lib().aipt_adamw_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
