"""ctypes binding of libba_hip.so (declarations in include/ba_hip.h).

The library is loaded lazily on first use and never replaced by a Python or
CPU implementation: if it is missing the call raises RuntimeError, exactly like
the reference's stub module does when its extension is not compiled
(src/blast3r/extensions/cujac/__init__.py:7-16).
"""
import ctypes
import os
import threading

import torch
from torch.autograd import forward_ad

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, 'libba_hip.so')

_lib = None
_lock = threading.Lock()

c_int = ctypes.c_int32
c_i64 = ctypes.c_int64
c_f = ctypes.c_float
c_d = ctypes.c_double
c_p = ctypes.c_void_p


class BaHuber(ctypes.Structure):
    _fields_ = [('weight_z', c_f), ('pnorm', c_f), ('max_pix_err', c_f), ('huber_delta', c_f),
                ('w_pts_null', c_f), ('is_depth_log', c_int)]


class BaLayout(ctypes.Structure):
    _fields_ = [('d', c_int), ('C', c_int), ('off_tau', c_int), ('off_zcf', c_int), ('hasK', c_int), ('hasP', c_int),
                ('hasZ', c_int), ('no_grad_f_from_rz', c_int), ('optim_Z0', c_int), ('optim_Z_1st_cam', c_int),
                ('wmin', c_f), ('wmax', c_f), ('dampen', c_d), ('adaptive', c_int), ('x_off', c_int)]


_LIN_FIELDS = [
    ('infos', c_p), ('n_imgs', c_int),
    ('chunk_obs', c_p), ('chunk_meta', c_p), ('slot_info', c_p),
    ('ct_pid', c_p), ('ct_first', c_p), ('ct_m', c_p), ('ct_mask', c_p),
    ('b_chunk_ptr', c_p), ('b_imgs', c_p), ('b_nimgs', c_p), ('b_slot_ptr', c_p), ('slot_pair', c_p),
    ('L', c_int),
    ('s_pix', c_p), ('s_std', c_p), ('s_dep', c_p), ('s_pid', c_p), ('s_img', c_p),
    ('K', c_p), ('P_rig2cam', c_p), ('P_rig2cam_stride', c_i64), ('P_w2rig', c_p), ('z_coefs', c_p), ('pts3d', c_p),
    ('enK', c_p), ('enP', c_p), ('enZ', c_p), ('enX', c_p),
    ('hp', BaHuber), ('lay', BaLayout),
    ('Hpp', c_p), ('gp', c_p), ('chunk_max', c_p), ('lam_p', c_p),
    ('partials', c_p), ('img_partials', c_p),
    ('dc', c_p), ('umap', c_p), ('dX', c_p), ('dX64', c_p),
    ('n_chunks', c_i64), ('n_batches', c_i64), ('n_pairs', c_i64),
    ('pair_ptr', c_p), ('pair_src', c_p), ('img_ptr', c_p), ('img_src', c_p),
    ('S_pairs', c_p), ('e_img', c_p), ('dg_img', c_p),
    ('r_in', c_p), ('w_in', c_p), ('r_s0', c_i64), ('r_s1', c_i64), ('w_s0', c_i64), ('w_s1', c_i64),
    ('ct_pt', c_p), ('n_ctracks', c_i64), ('core', c_p),
    ('chunk_slots', c_p), ('chunk_ent', c_p), ('chunk_eptr', c_p), ('b_pos_slot', c_p), ('pfac', c_p),
    ('b_order', c_p), ('work_ctr', c_p), ('dc_img', c_p), ('real32', c_int),
    ('parts', c_int), ('n_slots', c_i64),
]


class BaLinArgs(ctypes.Structure):
    _fields_ = _LIN_FIELDS


class BaPcgArgs(ctypes.Structure):
    _fields_ = [('n_u', c_i64), ('n_imgs', c_int), ('d', c_int), ('umap', c_p), ('inv_ptr', c_p), ('inv_src', c_p),
                ('leaf', c_p), ('row_ptr', c_p), ('row_ent', c_p), ('pair_i1', c_p), ('pair_i2', c_p),
                ('S_pairs', c_p), ('e_img', c_p), ('dg_img', c_p), ('dampen', c_d), ('adaptive', c_int),
                ('maxiter', c_int), ('tol', c_d),
                ('rhs', c_p), ('diagA', c_p), ('damp', c_p), ('x', c_p), ('xbest', c_p), ('r', c_p), ('z', c_p),
                ('p', c_p), ('y_img', c_p), ('partials', c_p), ('state', c_p), ('istate', c_p),
                ('S_rows', c_p), ('n_row_ent', c_i64), ('row_u', c_p), ('long_u', c_p), ('n_long', c_i64),
                ('long_ptr', c_p), ('long_idx', c_p), ('img_part', c_p), ('src1', c_p), ('long_rng', c_p),
                ('row_cap', c_int), ('real32', c_int)]

class BaPcgPairs(ctypes.Structure):
    _fields_ = [('t', c_p), ('p_img', c_p), ('up_ptr', c_p), ('n_pairs', c_i64)]


class BaPcgResident(ctypes.Structure):
    _fields_ = [('words', c_p), ('shared_u', c_p), ('n_shared', c_int), ('m', c_int), ('max_blk', c_int),
                ('max_col', c_int), ('limit', c_i64)]


class BaPmArgs(ctypes.Structure):
    _fields_ = [('infos', c_p), ('n_imgs', c_int), ('n_tracks', c_int),
                ('run_ptr', c_p), ('run_obs', c_p), ('run_trk', c_p), ('run_img', c_p), ('img_run_ptr', c_p),
                ('trk_run_ptr', c_p), ('trk_run', c_p), ('trk_obs_ptr', c_p), ('trk_obs', c_p), ('obs_img', c_p),
                ('pair_i1', c_p), ('pair_i2', c_p), ('diag_pair', c_p), ('term_ptr', c_p), ('term', c_p),
                ('pair_sched', c_p), ('n_obs', c_i64), ('n_runs', c_i64), ('n_pairs', c_i64),
                ('pids', c_p), ('pix2d', c_p), ('pix2d_std', c_p), ('pix2d_dep', c_p),
                ('K', c_p), ('P_rig2cam', c_p), ('P_rig2cam_stride', c_i64), ('P_w2rig', c_p), ('z_coefs', c_p),
                ('pts3d', c_p), ('enK', c_p), ('enP', c_p), ('enZ', c_p), ('enX', c_p),
                ('hp', BaHuber), ('lay', BaLayout),
                ('r_in', c_p), ('w_in', c_p), ('r_s0', c_i64), ('r_s1', c_i64), ('w_s0', c_i64), ('w_s1', c_i64),
                ('pobs', c_p), ('wobs', c_p), ('jslots', c_p), ('vslots', c_p), ('yrun', c_p), ('Hpp', c_p), ('gp', c_p), ('tmax', c_p), ('lam_p', c_p), ('pfac', c_p), ('V', c_p),
                ('S_pairs', c_p), ('e_img', c_p), ('dg_img', c_p), ('dc_img', c_p), ('dX', c_p), ('dX64', c_p),
                ('real32', c_int), ('n_terms', c_i64)]


class BaCholArgs(ctypes.Structure):
    _fields_ = [('mode', c_int), ('A', c_p), ('lda', c_i64), ('Linv', c_p), ('pair_idx', c_p), ('kind', c_p),
                ('shared_u', c_p), ('n_shared', c_int), ('w', c_int), ('db', c_int), ('bcol', c_p), ('bpos', c_p),
                ('n_pairs', c_i64), ('info', c_p),
                ('work', c_p)]


PCG_LONG_LIST = 32          # BA_PCG_LONG_LIST in include/ba_hip.h
PCG_BLOCK = 256             # unknowns per block of the PCG update launch (long_ptr granularity)


class BaSampleArgs(ctypes.Structure):
    _fields_ = [('map_addr', c_p), ('map_hw', c_p), ('H', c_int), ('W', c_int), ('Cm', c_int), ('pix_stride', c_int),
                ('insert_ones', c_int),
                ('cum_nppi', c_p), ('n_imgs', c_i64), ('pix2d', c_p), ('n_obs', c_i64), ('out', c_p)]


class BaObsSet(ctypes.Structure):
    _fields_ = [('pids', c_p), ('pix2d', c_p), ('pix2d_std', c_p), ('pix2d_dep', c_p), ('nppi', c_p), ('n_imgs', c_i64)]


class BaGatherArgs(ctypes.Structure):
    _fields_ = [('a', BaObsSet), ('b', BaObsSet), ('sel_a', c_p), ('sel_b', c_p), ('pid_shift_b', c_int), ('C', c_int),
                ('n_out', c_i64), ('n_rows', c_i64), ('pids', c_p), ('pix2d', c_p), ('pix2d_std', c_p),
                ('pix2d_dep', c_p), ('nppi', c_p), ('total', c_p), ('workspace', c_p)]


class BaRemoveArgs(ctypes.Structure):
    _fields_ = [('in_', BaObsSet), ('n_rows', c_i64), ('n_tracks', c_i64), ('C', c_int), ('bad_int64', c_int),
                ('bad', c_p), ('n_bad', c_i64), ('pids', c_p), ('pix2d', c_p), ('pix2d_std', c_p), ('pix2d_dep', c_p),
                ('nppi', c_p), ('old_to_keep', c_p), ('counts', c_p), ('workspace', c_p)]


class BaTangentArgs(ctypes.Structure):
    _fields_ = [('depth_addr', c_p), ('ref_addr', c_p), ('map_hw', c_p), ('H', c_int), ('W', c_int),
                ('depth_pix_stride', c_int), ('ref_pix_stride', c_int), ('K', c_p), ('cam_ids', c_p), ('z_coefs', c_p),
                ('n_imgs', c_i64), ('C', c_int), ('tan_stride', c_int), ('normalize', c_int), ('optim_Z0', c_int),
                ('fp64', c_int), ('compute_gn', c_int), ('weight', c_d), ('eps', c_d), ('loss', c_p), ('g_z', c_p),
                ('H_z', c_p), ('workspace', c_p), ('workspace_bytes', c_i64)]


class BaRotaryArgs(ctypes.Structure):
    # the header's arrays of two, element by element
    _fields_ = [('x0', c_p), ('x1', c_p), ('y0', c_p), ('y1', c_p),
                ('x_sb0', c_i64), ('x_sb1', c_i64), ('x_st0', c_i64), ('x_st1', c_i64), ('x_sh0', c_i64), ('x_sh1', c_i64),
                ('y_sb0', c_i64), ('y_sb1', c_i64), ('y_st0', c_i64), ('y_st1', c_i64), ('y_sh0', c_i64), ('y_sh1', c_i64),
                ('heads0', c_int), ('heads1', c_int), ('n_x', c_int),
                ('dtype', c_int), ('B', c_i64), ('T', c_i64), ('dim', c_int), ('part', c_int), ('axes', c_int),
                ('interleaved', c_int), ('inverse', c_int), ('pos_int64', c_int), ('positions', c_p),
                ('pos_sb', c_i64), ('pos_st', c_i64), ('pos_sa', c_i64), ('turns', c_p), ('factor', c_f)]


class BaKvArgs(ctypes.Structure):
    _fields_ = [('k', c_p), ('v', c_p), ('scales', c_p), ('n_blocks', c_i64), ('heads', c_int), ('dim', c_int),
                ('bits', c_int), ('n_seqs', c_int), ('pages', c_p), ('pages_stride', c_i64), ('n_pages', c_int),
                ('dtype', c_int), ('starts', c_p), ('offsets', c_p), ('n_rows', c_i64), ('rows_per_seq', c_i64),
                ('max_rows', c_i64), ('rk', c_p), ('rv', c_p), ('rk_st', c_i64), ('rk_sh', c_i64), ('rv_st', c_i64),
                ('rv_sh', c_i64)]


class BaKvAttendArgs(ctypes.Structure):
    _fields_ = [('k', c_p), ('v', c_p), ('scales', c_p), ('n_blocks', c_i64), ('heads', c_int), ('dim', c_int),
                ('bits', c_int), ('n_seqs', c_int), ('pages', c_p), ('pages_stride', c_i64), ('n_pages', c_int),
                ('dtype', c_int), ('lengths', c_p), ('offsets', c_p), ('n_rows', c_i64), ('rows_per_seq', c_i64),
                ('max_rows', c_i64), ('q', c_p), ('o', c_p), ('lse', c_p), ('q_st', c_i64), ('q_sh', c_i64),
                ('o_st', c_i64), ('o_sh', c_i64), ('q_heads', c_int), ('causal', c_int), ('window', c_i64),
                ('scale', c_f), ('n_splits', c_int), ('workspace', c_p), ('workspace_bytes', c_i64)]


class BaKvScoredArgs(BaKvAttendArgs):
    # the header's struct begins with ba_kv_attend_args, whose size is a multiple of what follows
    _fields_ = [('slopes', c_p), ('prefix', c_p), ('since', c_p), ('until', c_p), ('cap', c_f), ('shared', c_int),
                ('shared_parts', c_int), ('tile', c_int), ('shared_tile', c_int), ('reserved', c_int)]


class BaKvPool(ctypes.Structure):
    _fields_ = [('counts', c_p), ('used', c_p), ('marks', c_p), ('n_blocks', c_i64)]


class BaKvTable(ctypes.Structure):
    _fields_ = [('pages', c_p), ('stride', c_i64), ('n_seqs', c_int), ('n_pages', c_int)]


class BaKvCountArgs(ctypes.Structure):
    _fields_ = [('pool', BaKvPool), ('tables', ctypes.POINTER(BaKvTable)), ('n_tables', c_int), ('reserved', c_int)]


class BaKvFreeArgs(ctypes.Structure):
    _fields_ = [('pool', BaKvPool), ('free', c_p)]


class BaKvForkArgs(ctypes.Structure):
    _fields_ = [('pool', BaKvPool), ('from_', BaKvTable), ('to', BaKvTable), ('from_lengths', c_p), ('to_lengths', c_p),
                ('parents', c_p), ('children', c_p), ('n', c_int), ('reserved', c_int)]


class BaKvTrimArgs(ctypes.Structure):
    _fields_ = [('pool', BaKvPool), ('table', BaKvTable), ('first', c_p), ('last', c_p), ('rows', c_p), ('lengths', c_p),
                ('n_rows', c_int), ('all', c_int)]


class BaKvGrowArgs(ctypes.Structure):
    _fields_ = [('pool', BaKvPool), ('table', BaKvTable), ('lengths', c_p), ('more', c_p), ('each', c_int), ('max_new', c_int),
                ('src', c_p), ('dst', c_p), ('n', c_p), ('missing', c_p)]


class BaKvCompactArgs(ctypes.Structure):
    _fields_ = [('pool', BaKvPool), ('tables', ctypes.POINTER(BaKvTable)), ('n_tables', c_int), ('most', c_int), ('src', c_p),
                ('dst', c_p), ('n', c_p)]


class BaKvCopyArgs(ctypes.Structure):
    _fields_ = [('k', c_p), ('v', c_p), ('scales', c_p), ('n_blocks', c_i64), ('heads', c_int), ('dim', c_int), ('src', c_p),
                ('dst', c_p), ('count', c_p), ('n', c_int), ('reserved', c_int)]


# name -> (restype, argtypes)
_SIGS = {
    'ba_last_error': (ctypes.c_char_p, []),
    'ba_version': (c_int, []),
    'ba_residuals': (c_int, [c_p, c_int, c_p, c_p, c_i64, c_p, c_p, c_p, c_p, c_p, c_p, c_p, c_i64, c_int, c_int,
                             c_f, c_f, c_f, c_f, c_f, c_p, c_p]),
    'ba_jacobians': (c_int, [c_p, c_int, c_p, c_p, c_i64, c_p, c_p, c_p, c_p, c_p, c_p, c_i64, c_int, c_int, c_int,
                             c_p, c_p, c_p, c_p]),
    'ba_chol3x3_solve': (c_int, [c_p, c_p, c_p, c_i64, c_d, c_int, c_p]),
    'ba_blockcoo_workspace_size': (c_i64, [c_i64, c_i64]),
    'ba_blockcoo_matvec': (c_int, [c_p, c_int, c_int, c_p, c_p, c_int, c_i64, c_p, c_p, c_i64, c_i64, c_int, c_int,
                                   c_p, c_i64, c_p]),
    'ba_einsum_bki_bkj': (c_int, [c_p, c_i64, c_i64, c_p, c_i64, c_i64, c_p, c_i64, c_int, c_int, c_int, c_int, c_p]),
    'ba_exp_se3': (c_int, [c_p, c_p, c_i64, c_p]),
    'ba_plan_create': (c_p, [c_p, c_int, c_p, c_i64, c_int, c_int, c_int, c_i64]),
    'ba_plan_query': (c_int, [c_p, c_p, c_p]),
    'ba_plan_export': (c_int, [c_p, c_int, c_p]),
    'ba_plan_destroy': (None, [c_p]),
    'ba_plan_last_error': (ctypes.c_char_p, []),
    'ba_pm_dplan_create': (c_p, [c_p, c_int, c_p, c_i64, c_int, c_p]),
    'ba_pm_dplan_query': (c_int, [c_p, c_p, c_p]),
    'ba_pm_dplan_array': (c_p, [c_p, c_int]),
    'ba_pm_dplan_copy': (c_int, [c_p, c_int, c_p, c_p]),
    'ba_pm_dplan_destroy': (None, [c_p]),
    'ba_pm_dplan_last_error': (ctypes.c_char_p, []),
    'ba_plan_append': (c_p, [c_p, c_p, c_int, c_p, c_i64, c_int]),
    'ba_plan_array': (c_p, [c_p, c_int]),
    'ba_plan_stable': (c_int, [c_p, c_p, c_p]),
    'ba_plan_shift_ids': (c_int, [c_p, c_p, c_p, c_i64, c_p]),
    'ba_abi_sizeof': (c_i64, [ctypes.c_char_p]),
    'ba_linearize_schur': (c_int, [ctypes.POINTER(BaLinArgs), c_p]),
    'ba_linearize_stage': (c_int, [ctypes.POINTER(BaLinArgs), c_int, c_p]),
    'ba_backsubstitute': (c_int, [ctypes.POINTER(BaLinArgs), c_p]),
    'ba_pcg_solve': (c_int, [ctypes.POINTER(BaPcgArgs), c_p]),
    'ba_pcg_solve_range': (c_int, [ctypes.POINTER(BaPcgArgs), ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, c_p,
                                   c_p]),
    'ba_pcg_solve_pairs_range': (c_int, [ctypes.POINTER(BaPcgArgs), ctypes.POINTER(BaPcgPairs), ctypes.c_int32,
                                         ctypes.c_int32, ctypes.c_int32, c_p, c_p]),
    'ba_pcg_resident_plan': (ctypes.c_int32, [c_p, c_int, c_int, c_int, c_int, c_int, c_p, c_p]),
    'ba_pcg_resident_words': (c_i64, [c_int, c_int, c_int, c_int]),
    'ba_pcg_solve_resident': (c_int, [ctypes.POINTER(BaPcgArgs), ctypes.POINTER(BaPcgResident), c_p]),
    'ba_host_mapped_ptr': (c_p, [c_p]),
    'ba_pcg_partials_size': (c_i64, [c_i64]),
    'ba_apply_update': (c_int, [c_p, c_p, c_p, c_p, c_p, c_p, c_p, c_p, c_f, c_f, c_int, c_int, c_int, c_int, c_i64,
                                c_p, c_p, c_p, c_p, c_p]),
    'ba_objective_workspace_bytes': (c_i64, [c_i64]),
    'ba_objective': (c_int, [c_p, c_i64, c_int, c_p, c_p, c_p]),
    'ba_objective_noalloc': (c_int, [c_p, c_i64, c_int, c_p, c_p]),
    'ba_chol_dense_lda': (c_i64, [c_i64]),
    'ba_pm_plan_create': (c_p, [c_p, c_int, c_p, c_i64, c_int]),
    'ba_pm_plan_query': (c_int, [c_p, c_p, c_p]),
    'ba_pm_plan_export': (c_int, [c_p, c_int, c_p]),
    'ba_pm_plan_destroy': (None, [c_p]),
    'ba_schur_parts': (ctypes.c_int32, [c_i64, c_i64, c_i64, ctypes.c_int32]),
    'ba_pm_linearize_schur': (c_int, [ctypes.POINTER(BaPmArgs), c_p]),
    'ba_pm_linearize_stage': (c_int, [ctypes.POINTER(BaPmArgs), c_int, c_p]),
    'ba_pm_backsubstitute': (c_int, [ctypes.POINTER(BaPmArgs), c_p]),
    'ba_pm_slot_doubles': (c_i64, [c_i64, c_int, c_int]),
    'ba_chol_band_lds_bytes': (c_i64, [c_int, c_int, c_int]),
    'ba_chol_work_doubles': (c_i64, [c_int, c_i64, c_int, c_int, c_int, c_int]),
    'ba_chol_band_superblocks': (c_int, [c_int, c_int, c_int, c_int]),
    'ba_reduced_solve': (c_int, [ctypes.POINTER(BaPcgArgs), ctypes.POINTER(BaCholArgs), c_p]),
    'ba_nonfinite_flags': (c_int, [c_p, c_p, c_int, c_p, c_p]),
    'ba_stream_triad': (c_int, [c_p, c_p, c_p, ctypes.c_double, c_i64, c_p]),
    'ba_sample_depth': (c_int, [ctypes.POINTER(BaSampleArgs), c_p]),
    'ba_tracks_gather': (c_int, [ctypes.POINTER(BaGatherArgs), c_p]),
    'ba_tracks_remove': (c_int, [ctypes.POINTER(BaRemoveArgs), c_p]),
    'ba_tracks_to_dense': (c_int, [c_p, c_p, c_p, c_i64, c_i64, c_i64, c_i64, c_p, c_p, c_p]),
    'ba_tracks_img_id': (c_int, [c_p, c_i64, c_i64, c_p, c_p, c_p]),
    'ba_tracks_workspace_bytes': (c_i64, [c_i64, c_i64, c_i64]),
    'ba_tangent_prior': (c_int, [ctypes.POINTER(BaTangentArgs), c_p]),
    'ba_tangent_workspace_bytes': (c_i64, [c_i64, c_int, c_int, c_int, c_int, c_int, c_int]),
    'ba_planar_confidence': (c_int, [c_p, c_int, c_int, c_f, c_p, c_p]),
    'ba_add_z_prior': (c_int, [c_p, c_p, c_p, c_p, c_p, c_p, c_i64, c_int, c_int, c_int, c_p]),
    'ba_rotary': (c_int, [ctypes.POINTER(BaRotaryArgs), c_p]),
    'ba_kv_write': (c_int, [ctypes.POINTER(BaKvArgs), c_p]),
    'ba_kv_read': (c_int, [ctypes.POINTER(BaKvArgs), c_p]),
    'ba_kv_attend': (c_int, [ctypes.POINTER(BaKvAttendArgs), c_p]),
    'ba_kv_attend_splits': (c_int, [c_int, c_int, c_int, c_int, c_i64, c_int]),
    'ba_kv_attend_workspace_bytes': (c_i64, [c_i64, c_int, c_int, c_int]),
    'ba_kv_attend_scored': (c_int, [ctypes.POINTER(BaKvScoredArgs), c_p]),
    'ba_kv_scored_plan': (None, [ctypes.POINTER(BaKvScoredArgs)]),
    'ba_kv_pool_count': (c_int, [ctypes.POINTER(BaKvCountArgs), c_p]),
    'ba_kv_pool_free': (c_int, [ctypes.POINTER(BaKvFreeArgs), c_p]),
    'ba_kv_pool_fork': (c_int, [ctypes.POINTER(BaKvForkArgs), c_p]),
    'ba_kv_pool_trim': (c_int, [ctypes.POINTER(BaKvTrimArgs), c_p]),
    'ba_kv_pool_grow': (c_int, [ctypes.POINTER(BaKvGrowArgs), c_p]),
    'ba_kv_pool_compact': (c_int, [ctypes.POINTER(BaKvCompactArgs), c_p]),
    'ba_kv_copy': (c_int, [ctypes.POINTER(BaKvCopyArgs), c_p]),
}

EXPORTED = tuple(_SIGS)


ABI_STRUCTS = {'ba_huber': BaHuber, 'ba_layout': BaLayout, 'ba_lin_args': BaLinArgs, 'ba_pm_args': BaPmArgs,
               'ba_pcg_args': BaPcgArgs, 'ba_pcg_pairs': BaPcgPairs, 'ba_pcg_resident': BaPcgResident, 'ba_chol_args': BaCholArgs, 'ba_sample_args': BaSampleArgs,
               'ba_obs_set': BaObsSet, 'ba_gather_args': BaGatherArgs, 'ba_remove_args': BaRemoveArgs,
               'ba_tangent_args': BaTangentArgs, 'ba_rotary_args': BaRotaryArgs, 'ba_kv_args': BaKvArgs,
               'ba_kv_attend_args': BaKvAttendArgs, 'ba_kv_scored_args': BaKvScoredArgs, 'ba_kv_pool': BaKvPool,
               'ba_kv_table': BaKvTable, 'ba_kv_fork_args': BaKvForkArgs, 'ba_kv_trim_args': BaKvTrimArgs,
               'ba_kv_grow_args': BaKvGrowArgs, 'ba_kv_copy_args': BaKvCopyArgs, 'ba_kv_count_args': BaKvCountArgs,
               'ba_kv_compact_args': BaKvCompactArgs, 'ba_kv_free_args': BaKvFreeArgs}


def _check_abi(L):
    """Every argument struct here has the library's size (a field missing on one side would hand
    the kernels shifted pointers)."""
    bad = [(n, ctypes.sizeof(cls), int(L.ba_abi_sizeof(n.encode()))) for n, cls in ABI_STRUCTS.items()
           if ctypes.sizeof(cls) != int(L.ba_abi_sizeof(n.encode()))]
    if bad:
        raise RuntimeError(f'libba_hip.so struct layout differs from the Python binding: {bad}')


def lib():
    """The loaded library (raises RuntimeError when it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise RuntimeError(f'libba_hip.so is not built ({LIB_PATH}); run `python -m blast3r_amd.build` '
                                   'or __graft_entry__.build()')
            L = ctypes.CDLL(LIB_PATH)
            for name, (res, args) in _SIGS.items():
                f = getattr(L, name)
                f.restype = res
                f.argtypes = args
            _check_abi(L)
            _lib = L
    return _lib


def check(status):
    if status != 0:
        msg = lib().ba_last_error()
        raise RuntimeError((msg or b'libba_hip error').decode())


def stream_ptr(device=None):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)
_device = getattr(torch._C, '_cuda_getDevice', torch.cuda.current_device)       # there are tensors on it: it was started
_tracing = getattr(torch._C, '_is_tracing', torch.jit.is_tracing)
_modes = getattr(torch._C, '_len_torch_dispatch_stack', lambda: 1)


def _traced():
    """Whether a trace of torch's operations is being made, in which a launch would be missing."""
    if _tracing():
        return True
    from torch.fx.experimental.proxy_tensor import get_proxy_mode
    return get_proxy_mode() is not None


def launch(call, args, device):
    """One launch of ``call(args, stream)`` on the current stream of ``device``, as tensors on it expect (the short way
    for calls whose host time counts: no stream object, no device guard where the device is the current one)."""
    if (_tracing() or _modes()) and _traced():
        raise RuntimeError('a trace of torch operations cannot hold this call: it is a launch of libba_hip.so')
    index = device.index
    if _device() != index:
        with torch.cuda.device(index):
            return check(call(ctypes.byref(args), torch.cuda.current_stream(index).cuda_stream))
    stream = _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream
    status = call(ctypes.byref(args), stream)
    if status:
        check(status)


def dual_level():
    """Whether forward-mode tangents can be about (there are none outside a dual level)."""
    return getattr(forward_ad, '_current_level', 0) >= 0


def has_tangent(*tensors):
    """Whether one of them carries a tangent of forward-mode differentiation."""
    return dual_level() and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def overlaps(y, x):
    """Whether an output y cannot be written while x, of the same shape, is read: it has one place under several elements,
    or begins where x does with other strides.  (Views that overlap in other ways are not looked for.)"""
    if any(n > 1 and st == 0 for n, st in zip(y.shape, y.stride())):
        return True
    return y.data_ptr() == x.data_ptr() and any(n > 1 and a != b for n, a, b in zip(y.shape, y.stride(), x.stride()))


# written(tensors): a kernel wrote to tensors that were there before the call, so that what autograd or a cache keyed by
# versions keeps of them is out of date (without the public function's own 0.3 us)
written = getattr(torch._C, '_increment_version', torch.autograd.graph.increment_version)


def ptr(t):
    """Raw device pointer of a tensor (None -> NULL); a host tensor raises instead of handing a
    host address to a kernel."""
    if t is None:
        return None
    if not t.is_cuda:
        raise RuntimeError(f'expected a device tensor for a kernel argument, got one on {t.device}')
    return ctypes.c_void_p(t.data_ptr())
