"""ctypes binding of libyskn_b200.so (include/yskn_b200.h).

This mirrors how the reference's Python front end binds its native library
(python/yasakani/_native.py:26-39): a CDLL with declared argument types, integer
status codes and a thread-local error string. Device buffers are torch tensors
(plumbing only); every computation runs in the CUDA library. Import fails loudly
if the library has not been built; there is no fallback path.
"""
import ctypes as C
import os
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
LIB_PATH = os.path.join(PKG, "libyskn_b200.so")

OK, EINVAL, ECUDA, EOVERFLOW, ENONFINITE, ETIMEDOUT, ENOMEM = 0, -1, -2, -3, -4, -5, -6
LAYOUT_ROW, LAYOUT_WARP = 0, 1
LAYOUTS = {"row": LAYOUT_ROW, "warp": LAYOUT_WARP}
SIGN_RULES = {"splitmix64": 0, "mulberry32_7919_13": 1}

_vp, _i, _i64, _u64 = C.c_void_p, C.c_int, C.c_int64, C.c_uint64

_SIGNATURES = {
    "yskn_b200_last_error": (C.c_char_p, []),
    "yskn_b200_status": (_i, [_vp]),
    "yskn_repack_warp_to_frag": (_i, [_vp, _vp, _i, _i, _i, _vp]),
    "yskn_repack_warp_to_frag_host": (_i, [_vp, _vp, _i, _i, _i]),
    "yskn_b200_signs": (_i, [_i, _u64, _u64, _i64, _vp]),
    "yskn_b200_pack_bytes": (_i64, [_i, _i, _i]),
    "yskn_b200_pack": (_i, [_vp, _i, _i, _i, _i, _vp, _vp]),
    "yskn_b200_matrix_create": (_vp, [_vp, _i, _i, _i, _i, _i, _vp, _vp, _vp, _vp]),
    "yskn_b200_matrix_create_shard": (_vp, [_vp, _i, _i, _i, _i, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i]),
    "yskn_b200_matrix_destroy": (None, [_vp]),
    "yskn_b200_matrix_info": (_i, [_vp, _vp]),
    "yskn_b200_matrix_lut8": (_vp, [_vp]),
    "yskn_b200_matrix_tau": (_vp, [_vp]),
    "yskn_b200_matrix_signs_in": (_vp, [_vp]),
    "yskn_b200_matrix_signs_out": (_vp, [_vp]),
    "yskn_b200_weighted_sums": (_i, [_vp, _i, _vp, _vp, _i, _vp, _vp]),
    "yskn_b200_weighted_sums_prefix": (_i, [_vp, _vp, _vp, _i, _i, _vp, _vp]),
    "yskn_b200_weighted_sums_noalloc": (_i, [_vp, _i, _vp, _vp, _i, _vp, _vp]),
    "yskn_b200_quantize": (_i, [_vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp]),
    "yskn_b200_rescale": (_i, [_vp, _vp, _i, _i, _vp, _vp, _vp]),
    "yskn_b200_tp_create": (_vp, [_i, _i, _i, _vp]),
    "yskn_b200_tp_connect": (_i, [_vp, _vp]),
    "yskn_b200_tp_destroy": (None, [_vp]),
    "yskn_b200_tp_area": (_vp, [_vp]),
    "yskn_b200_tp_connect_peers": (_i, [_vp, _vp]),
    "yskn_b200_tp_set_wait": (_i, [_vp, C.c_double]),
    "yskn_b200_linear_rowpar": (_i, [_vp, _vp, _vp, _i, _vp, _vp, _vp]),
    "yskn_b200_restore": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _vp]),
    "yskn_b200_linear_work_bytes": (_i64, [_vp, _i, _i]),
    "yskn_b200_linear": (_i, [_vp, _i, _vp, _i, _vp, _vp, _vp, _vp]),
    "yskn_b200_kv4_attention_work_bytes": (_i64, [_i, _i, _i, _i]),
    "yskn_b200_kv4_attention": (_i, [_vp] * 9 + [_i] * 7 + [_vp] * 4),
    "yskn_b200_kv_encode": (_i, [_vp, _vp, _i, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _vp, _vp, _vp]),
    "yskn_b200_file_open": (_vp, [C.c_char_p]),
    "yskn_b200_file_close": (None, [_vp]),
    "yskn_b200_file_model_json": (C.c_char_p, [_vp]),
    "yskn_b200_file_tensor_count": (_i, [_vp]),
    "yskn_b200_file_vector_count": (_i, [_vp]),
    "yskn_b200_file_find": (_i, [_vp, C.c_char_p, _vp]),
    "yskn_b200_file_tensor_name": (C.c_char_p, [_vp, _i]),
    "yskn_b200_file_tensor_info": (_i, [_vp, _i, _vp]),
    "yskn_b200_file_vector_name": (C.c_char_p, [_vp, _i]),
    "yskn_b200_file_vector_info": (_i, [_vp, _i, _vp]),
    "yskn_b200_file_vector_read": (_i, [_vp, _i, _vp, _i64]),
    "yskn_b200_file_load_matrix": (_vp, [_vp, _i]),
    "yskn_b200_file_load_matrix_shard": (_vp, [_vp, _i, _i, _i, _i, _i]),
    "yskn_b200_embedding_create": (_vp, [_i, _vp, _vp, _i, _i, _vp, _vp, _vp]),
    "yskn_b200_embedding_destroy": (None, [_vp]),
    "yskn_b200_embedding_lookup": (_i, [_vp, _vp, _i, _vp, _vp]),
    "yskn_b200_file_load_embedding": (_vp, [_vp, _i, _i, _i]),
    "yskn_b200_residual_prepare": (_i, [_vp, _vp, _vp, _i, _i, C.c_float, _vp, _vp, _vp, _vp]),
    "yskn_b200_gated_product": (_i, [_vp, _vp, _i, _i, _vp, _vp]),
    "yskn_b200_head_select": (_i, [_vp, _i, _i, _vp, _vp, _vp, _vp]),
    "yskn_b200_attention_prep": (_i, [_vp] * 6 + [C.c_float, _i, _i, _i] + [_vp] * 5),
    "yskn_b200_gdn_gates": (_i, [_vp, _vp, _vp, _vp, _i, _i, _vp, _vp]),
    "yskn_b200_widen_bf16": (_i, [_vp, C.c_int64, _vp, _vp]),
    "yskn_b200_portable_math": (_i, [_i, _vp, C.c_int64, _vp, _vp, _vp]),
    "yskn_b200_linear_residual": (_i, [_vp] * 4 + [_i] + [_vp] * 8),
    "yskn_b200_linear_q8": (_i, [_vp, _i, _vp, _vp, _vp, C.c_float, _i, _vp, _vp, _vp]),
    "yskn_b200_gated_product_q8": (_i, [_vp, _vp, _i, _i, _vp, _vp, _vp, _vp]),
    "yskn_b200_gdn_step": (_i, [_vp] * 7 + [C.c_float, _i, _i, _vp, _vp, _vp, _vp]),
    "yskn_b200_matrix_create_rows": (_vp, [_vp, _i, _i, _i, _i, _i, _vp, _vp, _vp, _vp, _i, _vp, _i, _i]),
    "yskn_b200_gdn_gates_heads": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _vp, _vp]),
    "yskn_b200_gdn_step_heads": (_i, [_vp] * 7 + [C.c_float, _i, _i, _i, _i, _i, _i, _vp, _vp, _vp, _vp]),
    "yskn_b200_gdn_mixer": (_i, [_vp] * 4 + [_i] + [_vp] * 6 + [C.c_float, _i, _i, _vp, _vp, _vp, _vp]),
    "yskn_b200_gdn_mixer_heads": (_i, [_vp] * 4 + [_i] + [_vp] * 6 + [C.c_float, _i, _i, _i, _i, _i, _i, _vp, _vp,
                                                                        _vp, _vp]),
    "yskn_b200_linear_rowpar_residual": (_i, [_vp] * 5 + [_i] + [_vp] * 8),
    "yskn_b200_head_merge": (_i, [_vp, _vp, _i64, _vp, _i, _i, _vp, _vp, _vp, _vp]),
    "yskn_b200_linear_from_residual": (_i, [_vp, _i, _vp, _vp, _vp, _vp, C.c_float, _i, _vp, _vp, _vp, _vp]),
    "yskn_b200_linear_rowpar_q8": (_i, [_vp, _vp, _vp, _vp, _i, _vp, _vp]),
    "yskn_b200_batch_plan": (_i, [C.c_char_p, _vp]),
    "yskn_b200_paged_prep": (_i, [C.c_char_p, _vp]),
    "yskn_b200_prefix_attention_work_bytes": (_i64, [_i] * 6),
    "yskn_b200_prefix_attention": (_i, [C.c_char_p, _vp]),
    "yskn_b200_logits_adjust": (_i, [C.c_char_p, _vp]),
    "yskn_b200_tree_plan": (_i, [C.c_char_p, _vp]),
    "yskn_b200_tree_attention": (_i, [C.c_char_p, _vp]),
    "yskn_b200_tree_accept": (_i, [C.c_char_p, _vp]),
    "yskn_b200_batch_edit": (_i, [C.c_char_p, _vp]),
    "yskn_b200_cache_copy": (_i, [C.c_char_p, _vp]),
    "yskn_b200_cache_compact": (_i, [C.c_char_p, _vp]),
    "yskn_b200_token_logprobs": (_i, [C.c_char_p, _vp]),
}

_lib = None


class YsknError(RuntimeError):
    def __init__(self, code, message):
        super().__init__("%s (code %d)" % (message, code))
        self.code = code


def lib():
    """Load the library and declare every exported symbol of include/yskn_b200.h."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError("libyskn_b200.so is not built (run yasakani-for-mac_b200/build.py)")
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def exported_symbols():
    return sorted(_SIGNATURES)


def last_error():
    msg = lib().yskn_b200_last_error()
    return msg.decode() if msg else ""


def check(rc, what=""):
    if rc != OK:
        raise YsknError(rc, "%s: %s" % (what, last_error()))
    return rc


def _ptr(t):
    """A device tensor's address, or a raw device address given as an int."""
    if t is None:
        return None
    if isinstance(t, int):
        return C.c_void_p(t)
    return C.c_void_p(t.data_ptr())


def _stream(stream):
    if stream is None:
        import torch
        stream = torch.cuda.current_stream()
    return C.c_void_p(stream.cuda_stream)


def signs(rule, seed, offset, n):
    import numpy as np
    out = np.empty(n, np.int8)
    check(lib().yskn_b200_signs(SIGN_RULES[rule], seed, offset, n, out.ctypes.data), "signs")
    return out


class Matrix:
    """One compressed matrix on the device (yskn_b200_matrix_create)."""

    def __init__(self, d_codes, layout, rows, physical_rows, cols, bits, lut16, scale16, signs_in, signs_out=None,
                 shard=None):
        """shard: (row_begin, row_end, col_begin, col_end) of the whole tensor described by
        the other arguments (yskn_b200_matrix_create_shard), or None for the whole tensor;
        or ([(row_begin, row_end), ...], col_begin, col_end): several row ranges stored one
        after another (yskn_b200_matrix_create_rows)."""
        import numpy as np
        lut16 = np.ascontiguousarray(lut16, np.uint16)
        scale16 = np.ascontiguousarray(scale16, np.uint16)
        signs_in = np.ascontiguousarray(signs_in, np.int8)
        so = None if signs_out is None else np.ascontiguousarray(signs_out, np.int8)
        args = (_ptr(d_codes), LAYOUTS.get(layout, layout), rows, physical_rows, cols, bits, lut16.ctypes.data,
                scale16.ctypes.data, signs_in.ctypes.data, None if so is None else so.ctypes.data)
        if shard is None:
            h = lib().yskn_b200_matrix_create(*args)
            shard = (0, physical_rows, 0, cols)
        elif len(shard) == 3:
            ranges, c0, c1 = shard
            flat = (C.c_int * (2 * len(ranges)))(*[int(v) for r in ranges for v in r])
            h = lib().yskn_b200_matrix_create_rows(*args, len(ranges), flat, c0, c1)
        else:
            h = lib().yskn_b200_matrix_create_shard(*args, *shard)
        if not h:
            raise YsknError(EINVAL, "matrix_create: " + last_error())
        self.handle = C.c_void_p(h)
        self.shard = tuple(shard)
        if len(shard) == 3:
            ranges, c0, c1 = shard
            self.rows = sum(min(rows, r1) - r0 for r0, r1 in ranges)
            self.physical_rows = sum(r1 - r0 for r0, r1 in ranges)
        else:
            r0, r1, c0, c1 = shard
            self.rows, self.physical_rows = min(rows, r1) - r0, r1 - r0
        self.cols, self.bits = c1 - c0, bits
        self.has_rotation = so is not None

    @classmethod
    def _from_handle(cls, h, rows, physical_rows, cols, bits, has_rotation, shard):
        """A Matrix around a handle the library created (e.g. File.load_matrix)."""
        m = cls.__new__(cls)
        m.handle = C.c_void_p(h)
        r0, r1, c0, c1 = shard
        m.shard = tuple(shard)
        m.rows, m.physical_rows = min(rows, r1) - r0, r1 - r0
        m.cols, m.bits = c1 - c0, bits
        m.has_rotation = has_rotation
        return m

    def info(self):
        out = (C.c_int64 * 6)()
        check(lib().yskn_b200_matrix_info(self.handle, out), "matrix_info")
        return list(out)

    def close(self):
        if self.handle:
            lib().yskn_b200_matrix_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def signs_in_ptr(self):
        return lib().yskn_b200_matrix_signs_in(self.handle)


ROLES = ("body", "head", "embedding", "draft")
_RULE_NAMES = ("splitmix64", "mulberry32_7919_13")  # YSKN_SIGNS_* order


class File:
    """A `.yskn` container opened and checked by the library (yskn_b200_file_open):
    `model` (the header's model object), `tensors` and `vectors` (name -> descriptor with
    the format's defaults applied), `vector(name)` (f32 values) and `load_matrix(name)`
    (a Matrix whose codes, table, scales and signs come from the file)."""

    def __init__(self, path):
        import json
        h = lib().yskn_b200_file_open(os.fsencode(path))
        if not h:
            raise YsknError(EINVAL, last_error())
        self.handle = C.c_void_p(h)
        self.path = path
        self.model = json.loads(lib().yskn_b200_file_model_json(self.handle).decode("utf-8"))
        self.tensors, self.vectors = {}, {}
        info = (C.c_int64 * 17)()
        for i in range(lib().yskn_b200_file_tensor_count(self.handle)):
            check(lib().yskn_b200_file_tensor_info(self.handle, i, info), "file_tensor_info")
            v = list(info)
            rot = lambda r, seed, off: dict(rule=_RULE_NAMES[r], seed=seed, offset=off)
            name = lib().yskn_b200_file_tensor_name(self.handle, i).decode("utf-8")
            self.tensors[name] = dict(
                index=i, name=name, role=ROLES[v[0]], rows=v[1], cols=v[2], physical_rows=v[3], bits=v[4],
                layout="warp" if v[5] == LAYOUTS["warp"] else "row", stream_off=v[6], stream_bytes=v[7],
                lut_off=v[8], scale_off=v[9], rot_in=rot(v[10], v[11], v[12]),
                rot_out=rot(v[14], v[15], v[16]) if v[13] else None)
        vinfo = (C.c_int64 * 3)()
        for i in range(lib().yskn_b200_file_vector_count(self.handle)):
            check(lib().yskn_b200_file_vector_info(self.handle, i, vinfo), "file_vector_info")
            name = lib().yskn_b200_file_vector_name(self.handle, i).decode("utf-8")
            self.vectors[name] = dict(index=i, name=name, off=vinfo[0], n=vinfo[1],
                                      dtype="bf16" if vinfo[2] == 1 else "f16")

    def vector(self, name):
        import numpy as np
        v = self.vectors[name]
        out = np.empty(v["n"], np.float32)
        check(lib().yskn_b200_file_vector_read(self.handle, v["index"], out.ctypes.data, v["n"]), "file_vector_read")
        return out

    def load_matrix(self, name, shard=None):
        t = self.tensors[name]
        if shard is None:
            h = lib().yskn_b200_file_load_matrix(self.handle, t["index"])
            shard = (0, t["physical_rows"], 0, t["cols"])
        else:
            h = lib().yskn_b200_file_load_matrix_shard(self.handle, t["index"], *shard)
        if not h:
            raise YsknError(EINVAL, "file_load_matrix: " + last_error())
        return Matrix._from_handle(h, t["rows"], t["physical_rows"], t["cols"], t["bits"], t["rot_out"] is not None,
                                   shard)

    def load_embedding(self, main, res=None, res2=None):
        """An Embedding from the coded table `main` and up to two residual tables."""
        idx = [self.tensors[n]["index"] if n is not None else -1 for n in (main, res, res2)]
        h = lib().yskn_b200_file_load_embedding(self.handle, *idx)
        if not h:
            raise YsknError(EINVAL, "file_load_embedding: " + last_error())
        t = self.tensors[main]
        return Embedding._from_handle(h, t["rows"], t["cols"])

    def close(self):
        if self.handle:
            lib().yskn_b200_file_close(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Embedding:
    """Coded embedding rows on the device (yskn_b200_embedding_create / _lookup)."""

    def __init__(self, parts, rows, cols, signs_in):
        """parts: 1..3 tuples (d_codes, bits, lut16, scale16), the main table first; d_codes
        a device tensor holding the row-layout code stream; signs_in the main table's."""
        import numpy as np
        keep = [(np.ascontiguousarray(l, np.uint16), np.ascontiguousarray(s, np.uint16)) for _, _, l, s in parts]
        n = len(parts)
        codes = (C.c_void_p * n)(*[_ptr(c) for c, _, _, _ in parts])
        bits = (C.c_int * n)(*[b for _, b, _, _ in parts])
        luts = (C.c_void_p * n)(*[l.ctypes.data for l, _ in keep])
        scales = (C.c_void_p * n)(*[s.ctypes.data for _, s in keep])
        si = np.ascontiguousarray(signs_in, np.int8)
        h = lib().yskn_b200_embedding_create(n, codes, bits, rows, cols, luts, scales, si.ctypes.data)
        if not h:
            raise YsknError(EINVAL, "embedding_create: " + last_error())
        self.handle, self.rows, self.cols = C.c_void_p(h), rows, cols

    @classmethod
    def _from_handle(cls, h, rows, cols):
        e = cls.__new__(cls)
        e.handle, e.rows, e.cols = C.c_void_p(h), rows, cols
        return e

    def lookup(self, tokens, out, stream=None):
        """bf16 bits [M][cols] into `out` (a 16-bit device tensor) for int32 `tokens` [M]."""
        check(lib().yskn_b200_embedding_lookup(self.handle, _ptr(tokens), tokens.shape[0], _ptr(out), _stream(stream)),
              "embedding_lookup")

    def close(self):
        if self.handle:
            lib().yskn_b200_embedding_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def residual_prepare(hidden, projection, norm_weight, eps, inp, inv_rms, gate=None, stream=None):
    """hidden (bf16 bits, [M][cols], updated), projection (f32 or None), norm_weight (bf16
    bits [cols]) -> inp (f32 [M][cols]), inv_rms (f32 [M]), gate (bf16 bits or None)."""
    check(lib().yskn_b200_residual_prepare(_ptr(hidden), _ptr(projection), _ptr(norm_weight), hidden.shape[0],
                                           hidden.shape[1], eps, _ptr(inp), _ptr(inv_rms), _ptr(gate),
                                           _stream(stream)), "residual_prepare")


def gated_product(gate, up, out, stream=None):
    """out = bf16(bf16(silu(bf16(gate))) * bf16(up)) as f32, for f32 [M][n] gate and up."""
    check(lib().yskn_b200_gated_product(_ptr(gate), _ptr(up), gate.shape[0], gate.shape[1], _ptr(out),
                                        _stream(stream)), "gated_product")


def head_select(logits, token=None, top_logits=None, top_ids=None, stream=None):
    """Greedy token (int32 [M]) and top-8 (f32 / int32 [M][8]) of f32 logits [M][n]."""
    check(lib().yskn_b200_head_select(_ptr(logits), logits.shape[0], logits.shape[1], _ptr(token), _ptr(top_logits),
                                      _ptr(top_ids), _stream(stream)), "head_select")


def attention_prep(q, k, v, q_norm, k_norm, positions, eps, query, gate, k_rot, v_rot, stream=None):
    """q f32 [M][n_qh][512], k, v f32 [M][n_kvh][256], norms bf16 bits [256], positions
    int32 [M] -> query, gate (bf16 bits [M][n_qh][256]), k_rot, v_rot (f32 [M][n_kvh][256])."""
    check(lib().yskn_b200_attention_prep(_ptr(q), _ptr(k), _ptr(v), _ptr(q_norm), _ptr(k_norm), _ptr(positions), eps,
                                         q.shape[0], q.shape[1], k.shape[1], _ptr(query), _ptr(gate), _ptr(k_rot),
                                         _ptr(v_rot), _stream(stream)), "attention_prep")


def widen_bf16(src, out, stream=None):
    """out (f32) = the bf16 values of src (16-bit tensor), element count of src."""
    check(lib().yskn_b200_widen_bf16(_ptr(src), src.numel(), _ptr(out), _stream(stream)), "widen_bf16")


def gdn_gates(hidden, inv_rms, wb, wa, gates, stream=None):
    check(lib().yskn_b200_gdn_gates(_ptr(hidden), _ptr(inv_rms), _ptr(wb), _ptr(wa), hidden.shape[0], hidden.shape[1],
                                    _ptr(gates), _stream(stream)), "gdn_gates")


def gdn_gates_heads(hidden, inv_rms, wb, wa, gates, stream=None):
    """yskn_b200_gdn_gates_heads: the gates of the value heads whose rows wb, wa hold."""
    check(lib().yskn_b200_gdn_gates_heads(_ptr(hidden), _ptr(inv_rms), _ptr(wb), _ptr(wa), wb.shape[0],
                                          hidden.shape[0], hidden.shape[1], _ptr(gates), _stream(stream)),
          "gdn_gates_heads")


def gdn_step_heads(qkv, z, gates, conv_w, a_log, dt_bias, norm_w, eps, state, history, out, v_head0, qk_head0,
                   qk_channels, n_commit=None, stream=None):
    """yskn_b200_gdn_step_heads: the step of state.shape[0] value heads from v_head0, with
    the query/key channels of key heads from qk_head0 (qk_channels each)."""
    n_commit = qkv.shape[0] if n_commit is None else n_commit
    check(lib().yskn_b200_gdn_step_heads(_ptr(qkv), _ptr(z), _ptr(gates), _ptr(conv_w), _ptr(a_log), _ptr(dt_bias),
                                         _ptr(norm_w), eps, qkv.shape[0], n_commit, state.shape[0], v_head0,
                                         qk_head0, qk_channels, _ptr(state), _ptr(history), _ptr(out),
                                         _stream(stream)), "gdn_step_heads")


def head_merge(part_logits, part_ids, offsets, token=None, top_logits=None, top_ids=None, stream=None):
    """yskn_b200_head_merge: part_logits f32 / part_ids int32 [n_parts][M][8] (views whose
    first dimension may be strided, the other two dense), offsets the parts' first ids."""
    n_parts, M = part_logits.shape[0], part_logits.shape[1]
    assert part_logits.stride(0) == part_ids.stride(0) and part_logits.stride(1) == 8 and part_ids.stride(1) == 8
    offs = (C.c_int32 * n_parts)(*[int(o) for o in offsets])
    check(lib().yskn_b200_head_merge(_ptr(part_logits), _ptr(part_ids), part_logits.stride(0), offs, n_parts, M,
                                     _ptr(token), _ptr(top_logits), _ptr(top_ids), _stream(stream)), "head_merge")


def gdn_step(qkv, z, gates, conv_w, a_log, dt_bias, norm_w, eps, state, history, out, n_commit=None, stream=None):
    """One Gated DeltaNet pass over qkv.shape[0] rows, committing after n_commit rows
    (default: all of them; 0 = provisional, state and history unchanged)."""
    n_commit = qkv.shape[0] if n_commit is None else n_commit
    check(lib().yskn_b200_gdn_step(_ptr(qkv), _ptr(z), _ptr(gates), _ptr(conv_w), _ptr(a_log), _ptr(dt_bias),
                                   _ptr(norm_w), eps, qkv.shape[0], n_commit, _ptr(state), _ptr(history), _ptr(out),
                                   _stream(stream)), "gdn_step")


def gdn_mixer(hidden, inv_rms, wb, wa, qkv, z, conv_w, a_log, dt_bias, norm_w, eps, state, history, out,
              n_commit=None, stream=None):
    """yskn_b200_gdn_mixer: gdn_gates then gdn_step (with the history) in one launch."""
    n_commit = qkv.shape[0] if n_commit is None else n_commit
    check(lib().yskn_b200_gdn_mixer(_ptr(hidden), _ptr(inv_rms), _ptr(wb), _ptr(wa), hidden.shape[1], _ptr(qkv),
                                    _ptr(z), _ptr(conv_w), _ptr(a_log), _ptr(dt_bias), _ptr(norm_w), eps,
                                    qkv.shape[0], n_commit, _ptr(state), _ptr(history), _ptr(out), _stream(stream)),
          "gdn_mixer")


def gdn_mixer_heads(hidden, inv_rms, wb, wa, qkv, z, conv_w, a_log, dt_bias, norm_w, eps, state, history, out,
                    v_head0, qk_head0, qk_channels, n_commit=None, stream=None):
    """yskn_b200_gdn_mixer_heads: gdn_gates_heads then gdn_step_heads in one launch."""
    n_commit = qkv.shape[0] if n_commit is None else n_commit
    check(lib().yskn_b200_gdn_mixer_heads(_ptr(hidden), _ptr(inv_rms), _ptr(wb), _ptr(wa), hidden.shape[1],
                                          _ptr(qkv), _ptr(z), _ptr(conv_w), _ptr(a_log), _ptr(dt_bias), _ptr(norm_w),
                                          eps, qkv.shape[0], n_commit, state.shape[0], v_head0, qk_head0,
                                          qk_channels, _ptr(state), _ptr(history), _ptr(out), _stream(stream)),
          "gdn_mixer_heads")


def _handles(mats):
    arr = (C.c_void_p * len(mats))(*[m.handle for m in mats])
    return arr


def weighted_sums(mats, act, scales, outs, stream=None):
    """int64 [M][physical_rows] per matrix (yskn_b200_weighted_sums)."""
    M = act.shape[0]
    outp = (C.c_void_p * len(outs))(*[o.data_ptr() for o in outs])
    check(lib().yskn_b200_weighted_sums(_handles(mats), len(mats), _ptr(act), _ptr(scales), M, outp, _stream(stream)),
          "weighted_sums")


def weighted_sums_noalloc(mats, act, scales, outs, stream=None):
    """yskn_b200_weighted_sums_noalloc: the same sums with the library allocating nothing
    (scratch in a static device array; M <= 64; calls on one device must not overlap)."""
    M = act.shape[0]
    outp = (C.c_void_p * len(outs))(*[o.data_ptr() for o in outs])
    check(lib().yskn_b200_weighted_sums_noalloc(_handles(mats), len(mats), _ptr(act), _ptr(scales), M, outp,
                                                _stream(stream)), "weighted_sums_noalloc")


def weighted_sums_prefix(mat, act, scales, n_rows, out, stream=None):
    check(lib().yskn_b200_weighted_sums_prefix(mat.handle, _ptr(act), _ptr(scales), act.shape[0], n_rows, _ptr(out),
                                               _stream(stream)), "weighted_sums_prefix")


def quantize(x, signs_dev_ptr, act, alpha, scales, row_quantum, stream=None):
    M, K = x.shape
    check(lib().yskn_b200_quantize(_ptr(x), signs_dev_ptr, M, K, _ptr(act), _ptr(alpha), _ptr(scales),
                                   _ptr(row_quantum), _stream(stream)), "quantize")


def rescale(alpha, row_max, scales, row_quantum, stream=None):
    """yskn_b200_rescale: the rows' integer grids from given row maxima of the group scales."""
    M, G = alpha.shape
    check(lib().yskn_b200_rescale(_ptr(alpha), _ptr(row_max), M, G, _ptr(scales), _ptr(row_quantum),
                                  _stream(stream)), "rescale")


TP_HANDLE_BYTES = 64


class TpExchange:
    """This rank's side of the row-parallel exchange (yskn_b200_tp_create / _connect):
    create, swap the handles between ranks (`connect(handles)` takes all of them in rank
    order), then pass it to linear_rowpar."""

    def __init__(self, world, rank, max_physical_rows):
        self._handle_buf = C.create_string_buffer(TP_HANDLE_BYTES)
        self.handle = lib().yskn_b200_tp_create(world, rank, max_physical_rows, self._handle_buf)
        if not self.handle:
            raise YsknError(-1, "tp_create: " + last_error())
        self.world, self.rank = world, rank

    @property
    def ipc_handle(self):
        return self._handle_buf.raw

    def connect(self, handles):
        blob = b"".join(handles)
        if len(blob) != TP_HANDLE_BYTES * self.world:
            raise ValueError("one %d-byte handle per rank expected" % TP_HANDLE_BYTES)
        check(lib().yskn_b200_tp_connect(self.handle, blob), "tp_connect")

    @property
    def area(self):
        """This rank's exchange area as a device address (yskn_b200_tp_area)."""
        return lib().yskn_b200_tp_area(self.handle)

    def connect_peers(self, areas):
        """Connect with the peers' areas given as device addresses in rank order (one
        process driving several devices); this rank's own entry is ignored."""
        if len(areas) != self.world:
            raise ValueError("one area per rank expected")
        arr = (C.c_void_p * self.world)(*[a or 0 for a in areas])
        check(lib().yskn_b200_tp_connect_peers(self.handle, arr), "tp_connect_peers")

    def set_wait(self, seconds):
        """Limit of each wait phase on the peers (yskn_b200_tp_set_wait)."""
        check(lib().yskn_b200_tp_set_wait(self.handle, float(seconds)), "tp_set_wait")

    def close(self):
        if self.handle:
            lib().yskn_b200_tp_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def linear_rowpar(exchange, mat, x_local, y, inv_rms=None, stream=None):
    """yskn_b200_linear_rowpar: the whole output of a row-parallel shard, on every rank."""
    check(lib().yskn_b200_linear_rowpar(exchange.handle, mat.handle, _ptr(x_local), x_local.shape[0], _ptr(inv_rms),
                                        _ptr(y), _stream(stream)), "linear_rowpar")


def linear_rowpar_q8(exchange, mat, act_local, alpha_local, y, stream=None):
    """yskn_b200_linear_rowpar_q8: the whole output of a row-parallel shard from this rank's
    int8 input columns, on every rank."""
    check(lib().yskn_b200_linear_rowpar_q8(exchange.handle, mat.handle, _ptr(act_local), _ptr(alpha_local),
                                           act_local.shape[0], _ptr(y), _stream(stream)), "linear_rowpar_q8")


def linear_rowpar_residual(exchange, mat, hidden, norm_weight, next_signs, act_out, alpha_out, bss_out, x=None,
                           act=None, alpha=None, gate_out=None, stream=None):
    """yskn_b200_linear_rowpar_residual: the row-parallel operator from this rank's input
    columns (x f32, or act/alpha int8) into the whole residual stream and next input."""
    M = (x if x is not None else act).shape[0]
    check(lib().yskn_b200_linear_rowpar_residual(exchange.handle, mat.handle, _ptr(x), _ptr(act), _ptr(alpha), M,
                                                 _ptr(hidden), _ptr(norm_weight), _ptr(next_signs), _ptr(act_out),
                                                 _ptr(alpha_out), _ptr(bss_out), _ptr(gate_out), _stream(stream)),
          "linear_rowpar_residual")


def restore(ws, row_quantum, inv_rms, mat, rotate_out, n_rows, clear_ws, y, stream=None):
    check(lib().yskn_b200_restore(_ptr(ws), _ptr(row_quantum), _ptr(inv_rms), mat.handle, ws.shape[0],
                                  int(rotate_out), n_rows, int(clear_ws), _ptr(y), _stream(stream)), "restore")


def linear_work_bytes(mats, M):
    return lib().yskn_b200_linear_work_bytes(_handles(mats), len(mats), M)


def linear(mats, x, work, ys, inv_rms=None, stream=None):
    yp = (C.c_void_p * len(ys))(*[y.data_ptr() for y in ys])
    check(lib().yskn_b200_linear(_handles(mats), len(mats), _ptr(x), x.shape[0], _ptr(inv_rms), _ptr(work), yp,
                                 _stream(stream)), "linear")


def linear_residual(mat, hidden, norm_weight, next_signs, act_out, alpha_out, bss_out, x=None, act=None,
                    alpha=None, gate_out=None, stream=None):
    """yskn_b200_linear_residual: restore `mat` from x (f32) or act/alpha (int8) into the
    residual stream `hidden` (bf16 as int16) and write the next operator's int8 input."""
    M = (x if x is not None else act).shape[0]
    check(lib().yskn_b200_linear_residual(mat.handle, _ptr(x), _ptr(act), _ptr(alpha), M, _ptr(hidden),
                                          _ptr(norm_weight), _ptr(next_signs), _ptr(act_out), _ptr(alpha_out),
                                          _ptr(bss_out), _ptr(gate_out), _stream(stream)), "linear_residual")


def linear_q8(mats, act, alpha, ys, bss=None, eps=0.0, inv_rms_out=None, stream=None):
    """yskn_b200_linear_q8: the operator from an int8 input (and block sums of squares)."""
    yp = (C.c_void_p * len(ys))(*[y.data_ptr() for y in ys])
    check(lib().yskn_b200_linear_q8(_handles(mats), len(mats), _ptr(act), _ptr(alpha), _ptr(bss), float(eps),
                                    act.shape[0], _ptr(inv_rms_out), yp, _stream(stream)), "linear_q8")


def linear_from_residual(mats, y_prev, hidden_in, hidden_out, norm_weight, eps, ys, gate_out=None, inv_rms_out=None,
                         stream=None):
    """yskn_b200_linear_from_residual: the operator whose input is the residual stream
    hidden_in plus the previous projection's rows y_prev, normalised (norm_weight, eps) and
    quantised in the launch; the updated stream goes to hidden_out."""
    yp = (C.c_void_p * len(ys))(*[y.data_ptr() for y in ys])
    check(lib().yskn_b200_linear_from_residual(_handles(mats), len(mats), _ptr(y_prev), _ptr(hidden_in),
                                               _ptr(hidden_out), _ptr(norm_weight), float(eps), y_prev.shape[0],
                                               _ptr(gate_out), _ptr(inv_rms_out), yp, _stream(stream)),
          "linear_from_residual")


def gated_product_q8(gate, up, signs, act, alpha, stream=None):
    """yskn_b200_gated_product_q8: the MLP product quantised for the down projection."""
    M, n = gate.shape
    check(lib().yskn_b200_gated_product_q8(_ptr(gate), _ptr(up), M, n, _ptr(signs), _ptr(act), _ptr(alpha),
                                           _stream(stream)), "gated_product_q8")


PORTABLE_FN = {"exp": 0, "exp2": 1, "log": 2, "log1p": 3, "sigmoid": 4, "silu": 5, "softplus": 6, "rsqrt": 7,
               "sincos": 8}


def portable_math(name, x, y, y2=None, stream=None):
    """yskn_b200_portable_math: the device portable function `name` over the f32 tensor x
    into y (sincos: cosine into y, sine into y2)."""
    check(lib().yskn_b200_portable_math(PORTABLE_FN[name], _ptr(x), x.numel(), _ptr(y), _ptr(y2), _stream(stream)),
          "portable_math")


def status(stream=None):
    return lib().yskn_b200_status(_stream(stream))


def repack_warp_to_frag(words, frag, rows, seqs, wps, stream=None):
    return lib().yskn_repack_warp_to_frag(_ptr(words), _ptr(frag), rows, seqs, wps, _stream(stream))


def pack(words, layout, physical_rows, cols, bits, out, stream=None):
    check(lib().yskn_b200_pack(_ptr(words), LAYOUTS.get(layout, layout), physical_rows, cols, bits, _ptr(out),
                               _stream(stream)), "pack")


def kv4_attention_work_bytes(M, n_query_heads, length, n_splits=0):
    return lib().yskn_b200_kv4_attention_work_bytes(M, n_query_heads, length, n_splits)


def kv4_attention(q, k_rows, k_scales, v_rows, v_scales, k_codebook, v_codebook, length, work, out, gate=None,
                  v_mean=None, attended=None, n_splits=0, kb=4, stream=None):
    """q, gate, out: bf16 [M][n_qh][256] (passed as int16/bfloat16 tensors); k_rows/v_rows:
    int32 [n_kvh][capacity][8*kb]; scales f32 [n_kvh][capacity]; codebooks bf16 [n_kvh][256]."""
    M, n_qh = q.shape[0], q.shape[1]
    n_kvh, capacity = k_rows.shape[0], k_rows.shape[1]
    check(lib().yskn_b200_kv4_attention(_ptr(q), _ptr(gate), _ptr(k_rows), _ptr(k_scales), _ptr(v_rows),
                                        _ptr(v_scales), _ptr(k_codebook), _ptr(v_codebook), _ptr(v_mean), M, n_qh,
                                        n_kvh, length, capacity, kb, n_splits, _ptr(work), _ptr(attended),
                                        _ptr(out), _stream(stream)), "kv4_attention")


def kv_encode(rows, row_group, tables, gains, mults, kb, vit2, words, scales, means=None, has_mean=None, dest=None,
              stream=None):
    """rows f32 [n][256]; row_group int32 [n]; tables int16 [groups][256]; gains f32 [groups];
    mults f32 [n_mult]; words int32 [*][8*kb]; scales f32 [*]; dest int64 [n] or None."""
    check(lib().yskn_b200_kv_encode(_ptr(rows), _ptr(row_group), rows.shape[0], _ptr(tables), _ptr(gains),
                                    _ptr(means), _ptr(has_mean), _ptr(mults), mults.shape[0], kb, int(vit2),
                                    _ptr(dest), _ptr(words), _ptr(scales), _stream(stream)), "kv_encode")


DT_F32, DT_F16, DT_BF16 = 0, 1, 2

# The batch operators take a struct of arguments (yskn_b200_*_args, in the header's order); packing
# one is ten times faster than converting as many ctypes arguments. The library reads the whole of it,
# so a format ends with the padding that C adds (0P: up to a pointer's alignment).
ARGS = {
    "batch_plan": struct.Struct("@3PqPP3P3P6i0P"),
    "paged_prep": struct.Struct("@3P6q2PqP2P3P3q10if128s0P"),
    "prefix_attention": struct.Struct("@P2qP2q2P3q2Pq2PPqP12if0P"),
    "logits_adjust": struct.Struct("@PqPq2P3P2PPqPq4i0P"),
    "tree_plan": struct.Struct("@5PqP3i0P"),
    "tree_attention": struct.Struct("@P2qP2q2P3q2Pq2PPqP12if0PPqi0P"),  # prefix_attention's, then the masks
    "tree_accept": struct.Struct("@6Pq3P3i0P"),
    "batch_edit": struct.Struct("@4PqPq5PqP6i0P"),
    "cache_copy": struct.Struct("@P3qPqP6i0P"),
    "cache_compact": struct.Struct("@P3qPq3Pq9i0P"),
    "token_logprobs": struct.Struct("@PqPq4P4i0P"),
}
_DT, _FN = {}, {}


def _types():
    import torch
    _DT.update({torch.float32: DT_F32, torch.float16: DT_F16, torch.bfloat16: DT_BF16, torch.int16: DT_BF16})
    _DT["i32"], _DT["i64"] = torch.int32, torch.int64
    _DT["device"] = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
    # the raw handle at once: building a torch.cuda.Stream object around it takes longer than a launch
    _DT["stream"] = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
        lambda device: torch.cuda.current_stream(device).cuda_stream)


def _dtype(t):
    """YSKN_DT_* of a tensor; int16 tensors hold bf16 bits, as everywhere in this binding."""
    d = _DT.get(t.dtype)
    if d is None:
        raise YsknError(EINVAL, "a tensor of f32, f16, bf16 or int16 (bf16 bits) expected, not %s" % t.dtype)
    return d


def _need(ok, what):
    if not ok:
        raise YsknError(EINVAL, what)


def _launch(name, packed, tensor, stream):
    """The call on `stream`, or on the current stream of the tensor's device."""
    fn = _FN.get(name)
    if fn is None:
        fn = _FN[name] = getattr(lib(), "yskn_b200_" + name)
    rc = fn(packed, stream.cuda_stream if stream is not None else _DT["stream"](tensor.get_device()))
    if rc:
        check(rc, name)


def batch_plan(lens, new_lens, block_tables, pool, free_count, block_size, lens_out, free_out, starts, slots, positions,
               requests, prefix_len=0, stream=None):
    """yskn_b200_batch_plan: blocks from `pool` (int32 stack of *free_count numbers) for the new
    tokens of each request (new_lens int32 [batch]; negative: the request has ended), written
    into block_tables (int32 [batch][width]); the new lengths and count, the served tokens
    before each request (starts int32 [batch + 1]) and per token its slot (int64), position
    and request (int32), -1 past the last one."""
    if not _DT:
        _types()
    i32 = _DT["i32"]
    B, width = block_tables.shape
    T, row = slots.numel(), block_tables.stride()
    _need(lens.dtype is i32 and new_lens.dtype is i32 and block_tables.dtype is i32 and pool.dtype is i32 and
          free_count.dtype is i32 and lens_out.dtype is i32 and free_out.dtype is i32 and starts.dtype is i32 and
          positions.dtype is i32 and requests.dtype is i32 and slots.dtype is _DT["i64"] and lens.numel() == B and
          new_lens.numel() == B and lens_out.numel() == B and starts.numel() == B + 1 and positions.numel() == T and
          requests.numel() == T and row[1] == 1 and free_count.numel() and free_out.numel() and
          lens.is_contiguous() and new_lens.is_contiguous() and pool.is_contiguous() and lens_out.is_contiguous() and
          starts.is_contiguous() and slots.is_contiguous() and positions.is_contiguous() and requests.is_contiguous(),
          "batch_plan: dense int32 arrays of the batch, int64 slots and as many positions and requests expected")
    _launch("batch_plan", ARGS["batch_plan"].pack(
        lens.data_ptr(), new_lens.data_ptr(), block_tables.data_ptr(), row[0], pool.data_ptr(), free_count.data_ptr(),
        lens_out.data_ptr(), free_out.data_ptr(), starts.data_ptr(), slots.data_ptr(), positions.data_ptr(),
        requests.data_ptr(), B, block_size, prefix_len, width, pool.numel(), T), lens, stream)


def paged_prep(q, k, v, slots, positions, query, k_cache, v_cache, inv_freq=None, axes=None, q_norm=None, k_norm=None,
               eps=1e-6, stream=None):
    """yskn_b200_paged_prep: q [T][n_qh][D], k and v [T][n_kvh][D] (f32 or the cache's type, any
    strides with dense channels) normalised (q_norm, k_norm bf16 [D]) and rotated (inv_freq f32
    [rot / 2], axes the position axis of each pair, positions int32 [n_axes][T] or [T]) into
    query (dense [T][n_qh][D]) and, at `slots` (int64 [T]), k_cache and v_cache (views
    [n_blocks][block_size][n_kvh][D] of the same strides)."""
    if not _DT:
        _types()
    shape, cache = query.shape, k_cache.shape
    T, n_qh, D = shape
    n_blocks, block_size, n_kvh, _ = cache
    qs, ks, vs, cs = q.stride(), k.stride(), v.stride(), k_cache.stride()
    src, dt = q.dtype, query.dtype
    _need(q.shape == shape and k.shape == (T, n_kvh, D) and v.shape == (T, n_kvh, D) and cache[3] == D and
          v_cache.shape == cache and v_cache.stride() == cs and cs[3] == 1 and qs[2] == 1 and ks[2] == 1 and
          vs[2] == 1 and query.is_contiguous(),
          "paged_prep: q, k, v of the caches' heads with dense channels, caches of one shape and strides expected")
    _need(k.dtype is src and v.dtype is src and k_cache.dtype is dt and v_cache.dtype is dt and
          slots.dtype is _DT["i64"] and slots.numel() == T and slots.is_contiguous(),
          "paged_prep: types of q, k, v or of the caches differ, or slots not dense int64")
    _need((q_norm is None or (_DT.get(q_norm.dtype) == DT_BF16 and q_norm.numel() == D and q_norm.is_contiguous())) and
          (k_norm is None or (_DT.get(k_norm.dtype) == DT_BF16 and k_norm.numel() == D and k_norm.is_contiguous())),
          "paged_prep: dense bf16 norms of a head's channels expected")
    rot = n_axes = stride = 0
    packed = b""
    if inv_freq is not None:
        rot = 2 * inv_freq.numel()
        ps = positions.shape
        n_axes, stride = (1, T) if len(ps) == 1 else (ps[0], positions.stride(0))
        packed = bytes(axes) if axes is not None else bytes(rot // 2)
        _need(positions.dtype is _DT["i32"] and ps[-1] == T and positions.stride(-1) == 1 and
              len(packed) == rot // 2 and len(packed) <= 128 and _DT.get(inv_freq.dtype) == DT_F32 and
              inv_freq.is_contiguous(),
              "paged_prep: int32 positions of every token, and a dense f32 frequency and an axis for each pair expected")
    _launch("paged_prep", ARGS["paged_prep"].pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], slots.data_ptr(),
        positions.data_ptr() if rot else 0, stride, inv_freq.data_ptr() if rot else 0,
        0 if q_norm is None else q_norm.data_ptr(), 0 if k_norm is None else k_norm.data_ptr(), query.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), cs[0], cs[1], cs[2], T, n_qh, n_kvh, D, rot, n_axes, n_blocks,
        block_size, _dtype(q), _dtype(query), eps, packed), query, stream)


def prefix_attention_work_bytes(tokens, batch, max_new, n_qh, n_kvh, head):
    n = lib().yskn_b200_prefix_attention_work_bytes(tokens, batch, max_new, n_qh, n_kvh, head)
    _need(n >= 0, "prefix_attention_work_bytes: unsupported shape")
    return n


def _attention_args(name, q, k_cache, v_cache, block_tables, lens, starts, max_new, work, out, prefix_blocks,
                    prefix_len, gate, scale):
    """The checked arguments of prefix_attention, as its struct has them."""
    if not _DT:
        _types()
    i32, dt = _DT["i32"], q.dtype
    shape, cache = out.shape, k_cache.shape
    T, n_qh, D = shape
    n_blocks, block_size, n_kvh, _ = cache
    B, width = block_tables.shape
    qs, cs, row = q.stride(), k_cache.stride(), block_tables.stride()
    # (not by _need: the messages would be put together at each call)
    if not (q.shape == shape and cache[3] == D and v_cache.shape == cache and v_cache.stride() == cs and cs[3] == 1 and
            qs[2] == 1 and out.is_contiguous() and k_cache.dtype is dt and v_cache.dtype is dt and out.dtype is dt):
        raise YsknError(EINVAL, name + ": q, out and caches of one type and head size with dense channels expected")
    if not (block_tables.dtype is i32 and lens.dtype is i32 and starts.dtype is i32 and lens.numel() == B and
            starts.numel() == B + 1 and row[1] == 1 and lens.is_contiguous() and starts.is_contiguous() and
            work.is_contiguous() and
            (not prefix_len or (prefix_blocks is not None and prefix_blocks.dtype is i32 and
                                prefix_blocks.is_contiguous() and prefix_blocks.numel() * block_size >= prefix_len))):
        raise YsknError(EINVAL, name + ": dense int32 tables, lengths and starts of one batch, and the prefix's blocks "
                        "expected")
    gs, gd = (0, 0), 0
    if gate is not None:
        gs, gd = gate.stride(), _dtype(gate)
        if not (gate.shape == shape and gs[2] == 1):
            raise YsknError(EINVAL, name + ": a gate of the queries' shape with dense channels expected")
    return (
        q.data_ptr(), qs[0], qs[1], 0 if gate is None else gate.data_ptr(), gs[0], gs[1], k_cache.data_ptr(),
        v_cache.data_ptr(), cs[0], cs[1], cs[2], prefix_blocks.data_ptr() if prefix_len else 0,
        block_tables.data_ptr(), row[0], lens.data_ptr(), starts.data_ptr(), work.data_ptr(),
        work.numel() * work.element_size(), out.data_ptr(), n_blocks, block_size, prefix_len, width, B, T, max_new,
        n_qh, n_kvh, D, _dtype(q), gd, D ** -0.5 if scale is None else scale)


def prefix_attention(q, k_cache, v_cache, block_tables, lens, starts, max_new, work, out, prefix_blocks=None,
                     prefix_len=0, gate=None, scale=None, stream=None):
    """yskn_b200_prefix_attention: q and gate (of q's type, or f32) [T][n_qh][D] with dense
    channels, the caches as paged_prep, each request's own blocks in block_tables (int32
    [batch][width]) and the shared prefix's in prefix_blocks; lens and starts as batch_plan writes them (at most max_new tokens
    a request) -> out (dense [T][n_qh][D]). scale defaults to 1 / sqrt(D). work: uint8, of
    prefix_attention_work_bytes(T, batch, max_new, n_qh, n_kvh, D) bytes."""
    _launch("prefix_attention", ARGS["prefix_attention"].pack(*_attention_args(
        "prefix_attention", q, k_cache, v_cache, block_tables, lens, starts, max_new, work, out, prefix_blocks,
        prefix_len, gate, scale)), out, stream)


def logits_adjust(logits, out, history=None, history_lens=None, prompt_lens=None, repetition=None, presence=None,
                  frequency=None, bias_ids=None, bias=None, mask=None, stream=None):
    """yskn_b200_logits_adjust: f32 logits [M][V] (dense rows, any row stride) -> out (may be
    logits). history int32 [M][L] with history_lens and prompt_lens int32 [M]; repetition,
    presence, frequency f32 [M]; bias_ids int32 and bias f32 [M][n] (dense); mask int32
    [M][>= ceil(V / 32)], a set bit for an allowed token."""
    if not _DT:
        _types()
    i32, f32 = _DT["i32"], logits.dtype
    shape, xs, os_ = logits.shape, logits.stride(), out.stride()
    M, V = shape
    _need(_dtype(logits) == DT_F32 and out.dtype is f32 and out.shape == shape and xs[1] == 1 and os_[1] == 1,
          "logits_adjust: f32 logits and output of one shape with dense rows expected")
    hs = ms = (0, 1)
    width = n_bias = hp = 0
    if history is not None:
        hs, (rows, width) = history.stride(), history.shape
        hp = history.data_ptr() or logits.data_ptr()  # one of no entries has no address, and is not read
        _need(history.dtype is i32 and rows == M and hs[1] == 1, "logits_adjust: int32 history rows expected")
    if mask is not None:
        ms, (rows, words) = mask.stride(), mask.shape
        _need(mask.dtype is i32 and rows == M and ms[1] == 1 and words * 32 >= V,
              "logits_adjust: int32 mask rows of a bit per token expected")
    _need((bias is None) == (bias_ids is None), "logits_adjust: a bias list needs its ids and values")
    if bias is not None:
        rows, n_bias = bias.shape
        _need(bias.dtype is f32 and bias_ids.dtype is i32 and bias_ids.shape == (rows, n_bias) and rows == M and
              bias.is_contiguous() and bias_ids.is_contiguous(), "logits_adjust: dense f32 biases of int32 ids expected")
    lp = pp = rp = ep = fp = 0
    ok = True
    if history_lens is not None:
        lp = history_lens.data_ptr()
        ok = history_lens.dtype is i32 and history_lens.numel() == M and history_lens.is_contiguous()
    if prompt_lens is not None:
        pp = prompt_lens.data_ptr()
        ok = ok and prompt_lens.dtype is i32 and prompt_lens.numel() == M and prompt_lens.is_contiguous()
    if repetition is not None:
        rp = repetition.data_ptr()
        ok = ok and repetition.dtype is f32 and repetition.numel() == M and repetition.is_contiguous()
    if presence is not None:
        ep = presence.data_ptr()
        ok = ok and presence.dtype is f32 and presence.numel() == M and presence.is_contiguous()
    if frequency is not None:
        fp = frequency.data_ptr()
        ok = ok and frequency.dtype is f32 and frequency.numel() == M and frequency.is_contiguous()
    _need(ok, "logits_adjust: a dense int32 length or f32 penalty for each row expected")
    _launch("logits_adjust", ARGS["logits_adjust"].pack(
        logits.data_ptr(), xs[0], hp, hs[0], lp, pp, rp, ep, fp,
        0 if bias is None else bias_ids.data_ptr(), 0 if bias is None else bias.data_ptr(),
        0 if mask is None else mask.data_ptr(), ms[0], out.data_ptr(), os_[0], M, V, width, n_bias), out, stream)


def _here(name, tensors):
    """All on the current device, which the call is launched on."""
    at = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != at:
            at = -1
    if at < 0 or at != _DT["device"]():
        raise YsknError(EINVAL, name + ": tensors on the current device expected")


def _flat(name, dtype, tensors):
    """The addresses of dense arrays of one type on the current device."""
    at, out = tensors[0].get_device(), []
    for t in tensors:
        if t.dtype is not dtype or not t.is_contiguous():
            raise YsknError(EINVAL, "%s: dense arrays of %s expected" % (name, dtype))
        if t.get_device() != at:
            at = -1
        out.append(t.data_ptr())
    if at < 0 or at != _DT["device"]():
        raise YsknError(EINVAL, name + ": tensors on the current device expected")
    return out


def tree_plan(parents, requests, starts, lens, mask, positions, stream=None):
    """yskn_b200_tree_plan: for each new token (parents int32 [T]: the new token of its request that it follows,
    negative for none; requests, starts and lens as batch_plan writes them) the bits of itself and its ancestors
    (mask int32 [T][words], a bit a new token of its request) and its position (int32 [T])."""
    if not _DT:
        _types()
    i32, T, B, (rows, words), row = _DT["i32"], parents.numel(), lens.numel(), mask.shape, mask.stride()
    if not (mask.dtype is i32 and mask.get_device() == parents.get_device() and rows == T and row[1] == 1 and
            requests.numel() == T and positions.numel() == T and starts.numel() == B + 1):
        raise YsknError(EINVAL, "tree_plan: int32 arrays of one batch and a mask row for each token expected")
    a, b, c, d, e = _flat("tree_plan", i32, (parents, requests, starts, lens, positions))
    _launch("tree_plan", ARGS["tree_plan"].pack(a, b, c, d, mask.data_ptr(), row[0], e, T, B, words), parents, stream)


def tree_attention(q, k_cache, v_cache, block_tables, lens, starts, max_new, mask, work, out, prefix_blocks=None,
                   prefix_len=0, gate=None, scale=None, stream=None):
    """yskn_b200_tree_attention: prefix_attention in which a new token sees, of its request's new rows, only
    those up to itself whose bit is set in its row of mask (int32 [T][words], as tree_plan writes it)."""
    args = _attention_args("tree_attention", q, k_cache, v_cache, block_tables, lens, starts, max_new, work, out,
                           prefix_blocks, prefix_len, gate, scale)
    (rows, words), row = mask.shape, mask.stride()
    _need(mask.dtype is _DT["i32"] and rows == q.shape[0] and row[1] == 1,
          "tree_attention: an int32 mask row for each token expected")
    used = [q, k_cache, v_cache, block_tables, lens, starts, mask, work, out]
    if prefix_len:
        used.append(prefix_blocks)
    if gate is not None:
        used.append(gate)
    _here("tree_attention", used)
    _launch("tree_attention", ARGS["tree_attention"].pack(*args, mask.data_ptr(), row[0], words), out, stream)


def tree_accept(tokens, parents, choice, starts, lens, path, accepted, lens_out, next_token, stream=None):
    """yskn_b200_tree_accept: of each request's tree (tokens and parents int32 [T]) the path that the model's choices
    (int32 [T], after each node) take: path (int32 [batch][width], -1 past its end), how many nodes it has,
    the lengths without the others' rows, and the choice after its last node (int32 [batch] each)."""
    if not _DT:
        _types()
    i32, T, B, (rows, width), row = _DT["i32"], tokens.numel(), lens.numel(), path.shape, path.stride()
    if not (path.dtype is i32 and path.get_device() == tokens.get_device() and rows == B and row[1] == 1 and
            parents.numel() == T and choice.numel() == T and starts.numel() == B + 1 and accepted.numel() == B and
            lens_out.numel() == B and next_token.numel() == B):
        raise YsknError(EINVAL, "tree_accept: int32 arrays of one batch and a path row for each request expected")
    a, b, c, d, e, f, g, h = _flat("tree_accept", i32, (tokens, parents, choice, starts, lens, accepted, lens_out,
                                                        next_token))
    _launch("tree_accept", ARGS["tree_accept"].pack(a, b, c, d, e, path.data_ptr(), row[0], f, g, h, B, T, width),
            tokens, stream)


def batch_edit(lens, keep, block_tables, pool, free_count, block_size, lens_out, free_out, source=None, tables_out=None,
               copies=None, n_copies=None, prefix_len=0, stream=None):
    """yskn_b200_batch_edit: request i keeps its first keep[i] rows, or becomes the first keep[i] rows of request
    source[i] (int32 [batch]; negative: it ends). Without a source the block tables stay valid; with one the new
    tables go to tables_out, and the blocks that cache_copy has to copy to copies (int32 [3][n]: block to read,
    block to write, rows) and their number to n_copies (int32 [1])."""
    if not _DT:
        _types()
    i32, (B, width), row = _DT["i32"], block_tables.shape, block_tables.stride()
    if not (block_tables.dtype is i32 and block_tables.get_device() == lens.get_device() and row[1] == 1 and
            lens.numel() == B and keep.numel() == B and lens_out.numel() == B and free_count.numel() and
            free_out.numel()):
        raise YsknError(EINVAL, "batch_edit: dense int32 arrays of the batch expected")
    a, b, c, d, e, f = _flat("batch_edit", i32, (lens, keep, pool, free_count, lens_out, free_out))
    if source is None:
        _launch("batch_edit", ARGS["batch_edit"].pack(a, b, 0, block_tables.data_ptr(), row[0], 0, 0, c, d, e, f, 0, 0,
                                                      0, B, block_size, prefix_len, width, pool.numel(), 0),
                lens, stream)
        return
    _need(tables_out is not None and copies is not None and n_copies is not None,
          "batch_edit: a source needs new tables, a list of copies and its count")
    ts, cs, (three, n) = tables_out.stride(), copies.stride(), copies.shape
    if not (tables_out.dtype is i32 and tables_out.shape == block_tables.shape and ts[1] == 1 and
            copies.dtype is i32 and three == 3 and cs[1] == 1 and source.numel() == B and n_copies.numel() and
            tables_out.get_device() == copies.get_device() == lens.get_device()):
        raise YsknError(EINVAL, "batch_edit: int32 source, tables of one shape and copies [3][n] expected")
    g, h = _flat("batch_edit", i32, (source, n_copies))
    _launch("batch_edit", ARGS["batch_edit"].pack(
        a, b, g, block_tables.data_ptr(), row[0], tables_out.data_ptr(), ts[0], c, d, e, f, copies.data_ptr(), cs[0],
        h, B, block_size, prefix_len, width, pool.numel(), n), lens, stream)


class CacheSet:
    """The K and V caches of a model's layers (16-bit views [n_blocks][block_size][n_kvh][D] of one shape and
    strides, as paged_prep takes them), for cache_copy and cache_compact. Keeps them alive."""

    def __init__(self, caches):
        caches = list(caches)
        _need(len(caches) > 0, "CacheSet: at least one cache expected")
        first = caches[0]
        _need(all(c.dim() == 4 and c.element_size() == 2 and c.dtype == first.dtype and c.shape == first.shape and
                  c.stride() == first.stride() and c.device == first.device for c in caches) and first.stride(3) == 1,
              "CacheSet: 16-bit caches of one type, shape, strides and device with dense channels expected")
        self.caches = caches
        self._pointers = (C.c_void_p * len(caches))(*[c.data_ptr() for c in caches])
        n_blocks, block_size, n_kvh, head = first.shape
        s = first.stride()
        self._head = (C.addressof(self._pointers), s[0], s[1], s[2])
        self._sizes = (len(caches), n_blocks, block_size, n_kvh, head)


def cache_copy(caches, copies, count=None, stream=None):
    """yskn_b200_cache_copy: in every cache of the CacheSet the blocks that batch_edit lists (copies int32 [3][n]:
    block to read, block to write, rows), the first *count (int32 [1]) of them or all."""
    if not _DT:
        _types()
    i32, (three, n), row = _DT["i32"], copies.shape, copies.stride()
    _need(copies.dtype is i32 and three == 3 and row[1] == 1 and
          (count is None or (count.dtype is i32 and count.numel())),
          "cache_copy: int32 copies [3][n] and a count expected")
    _here("cache_copy", (copies, caches.caches[0]) if count is None else (copies, caches.caches[0], count))
    _launch("cache_copy", ARGS["cache_copy"].pack(
        *caches._head, copies.data_ptr(), row[0], 0 if count is None else count.data_ptr(), *caches._sizes, n), copies,
        stream)


def cache_compact(caches, block_tables, lens, starts, path, prefix_len=0, stream=None):
    """yskn_b200_cache_compact: in every cache of the CacheSet, of each request's new rows (the last of its lens, as
    many as its starts say) those on its path (int32 [batch][width], as tree_accept writes it) made adjacent."""
    if not _DT:
        _types()
    i32, (B, width), (rows, nodes) = _DT["i32"], block_tables.shape, path.shape
    ts, ps = block_tables.stride(), path.stride()
    _need(block_tables.dtype is i32 and ts[1] == 1 and lens.numel() == B and starts.numel() == B + 1 and
          path.dtype is i32 and rows == B and ps[1] == 1,
          "cache_compact: int32 tables, lengths, starts and paths of one batch expected")
    _here("cache_compact", (block_tables, path, caches.caches[0]))
    a, b = _flat("cache_compact", i32, (lens, starts))
    _launch("cache_compact", ARGS["cache_compact"].pack(
        *caches._head, block_tables.data_ptr(), ts[0], a, b, path.data_ptr(), ps[0], *caches._sizes, B, width,
        prefix_len, nodes), lens, stream)


def token_logprobs(logits, tokens=None, logprobs=None, entropy=None, top_logprobs=None, top_ids=None, stream=None):
    """yskn_b200_token_logprobs: of f32 logits [M][V] (dense rows, any row stride) the log probabilities of tokens
    (int32 [M][n]) into logprobs (f32 [M][n]), the entropy (f32 [M]), and the most likely tokens into top_logprobs
    (f32 [M][k]) and top_ids (int32 [M][k]), k up to 32."""
    if not _DT:
        _types()
    i32, f32, (M, V), row = _DT["i32"], logits.dtype, logits.shape, logits.stride()
    n = k = stride = 0
    used = [logits]
    a = b = e = c = d = 0
    _need(_DT.get(f32) == DT_F32 and row[1] == 1, "token_logprobs: f32 logits with dense rows expected")
    _need((tokens is None) == (logprobs is None) and (top_ids is None) == (top_logprobs is None),
          "token_logprobs: tokens and their output, and both outputs of the most likely ones, go together")
    if tokens is not None:
        shape = tokens.shape
        (rows, n), (stride, step) = shape, tokens.stride()
        _need(tokens.dtype is i32 and rows == M and (step == 1 or n < 2) and logprobs.shape == shape and
              logprobs.dtype is f32 and logprobs.is_contiguous(),
              "token_logprobs: int32 tokens [M][n] and dense f32 log probabilities of their shape expected")
        used += (tokens, logprobs)
        a, b = tokens.data_ptr(), logprobs.data_ptr()
    if entropy is not None:
        _need(entropy.dtype is f32 and entropy.shape == (M,) and entropy.is_contiguous(),
              "token_logprobs: f32 entropy [M] expected")
        used.append(entropy)
        e = entropy.data_ptr()
    if top_ids is not None:
        shape = top_ids.shape
        rows, k = shape
        _need(rows == M and top_logprobs.shape == shape and top_ids.dtype is i32 and top_ids.is_contiguous() and
              top_logprobs.dtype is f32 and top_logprobs.is_contiguous(),
              "token_logprobs: dense int32 numbers and f32 log probabilities [M][k] expected")
        used += (top_logprobs, top_ids)
        c, d = top_logprobs.data_ptr(), top_ids.data_ptr()
    _here("token_logprobs", used)
    _launch("token_logprobs", ARGS["token_logprobs"].pack(logits.data_ptr(), row[0], a, stride, b, e, c, d, M, V, n, k),
            logits, stream)
