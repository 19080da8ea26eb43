"""Launch the hot kernels at the benchmark shapes, for rocprofv3.

    rocprofv3 --kernel-trace --stats -d OUT -- python3 -m fasth3inc_amd.profile_kernels gemv
    rocprofv3 --pmc FETCH_SIZE -d OUT -- python3 -m fasth3inc_amd.profile_kernels gemv
    rocprofv3 --pmc WRITE_SIZE -d OUT -- python3 -m fasth3inc_amd.profile_kernels copy

Workloads (each launch sequence is preceded by one untimed warmup launch):
  gemv   the six small-M shapes (M in {1,4,16}, K=5120, N in {5120,17408}):
         fh3_hip_matmul_prepared_dev -> k_gemv8 (M <= 4) and k_sweep
         (M = 16, after k_xprep), weights rotated over more than 256 MB of
         device copies so they come from HBM
  gemm   the DiT attention shapes (M=8192, K=5120, N in {15360,5120}):
         fh3_hip_matmul_prepared_dev -> k_wfrag, k_gemm256, and the activation
         prep k_xprep_r8
  mlp    the DiT MLP shapes (M=32768: up and gate K=5120 -> N=13824 with a
         2-decade per-super-block scale spread, down K=13824 -> N=5120 on
         SiLU-gated activations): fh3_hip_matmul_prepared_dev -> k_wfrag,
         k_gemm256, and the activation prep k_xprep_r8
  te     the text encoder's long Q4_K rows at M = 1 and 16 (o-projection
         K=8192 -> N=5120, down-projection K=25600 -> N=5120):
         fh3_hip_matmul_prepared_dev -> k_gemv8 (M = 1, K = 8192) or k_sweep in
         K slices then k_midm_sum; weights rotated as for gemv
  prompt 17 to 64 tokens at K = 5120 (M in {17, 32, 48, 64}, N in {5120,
         17408}): fh3_hip_matmul_prepared_dev -> k_sweep with two to four
         token blocks; weights rotated as for gemv
  mid    65, 128 and 256 tokens at K = 5120 (N in {5120, 17408}):
         fh3_hip_matmul_prepared_dev -> k_gemm with 128- or 256-token tiles
         and a K split, then k_midm_sum; weights rotated as for gemv
  single the 64 x 4096 x 4096 product of the reference's bench_matmul.c, one
         weight copy (warm in the Infinity Cache after the first launch, as the
         benchmark runs it): fh3_hip_matmul_prepared_dev -> k_skinny
  q56    Q5_K and Q6_K weights read in place at the text encoder's shapes
         (Q5_K 5120 -> 1024, Q6_K 5120 -> 1024, 8192 -> 5120, 25600 -> 5120)
         at M = 1, 16 and 300: fh3_hip_matmul_prepared_dev -> k_sweep<Q6_K>
         and k_skinny<Q5_K> (K slices / windows, then k_midm_sum, where they
         split K) and k_gemm<TBW, Q5_K / Q6_K> at 300; weights rotated as for
         gemv
  copy   hipMemcpy device-to-device of 256 MiB: a copy of known size that
         calibrates FETCH_SIZE / WRITE_SIZE against the bytes moved
  attn   the DiT attention branch at n = 16384 tokens, 40 heads of 128
         (hidden 5120): fh3_hip_attention_qkv_dev from a qkv projection
         output with q/k rmsnorm and rope3 on 96 channels -> k_attn_prep,
         k_attn_fwd
  vsa    video sparse attention at the reference CLI's 1024x576, 73-frame
         shape (6 text + 244 audio tokens, video grid 22x18x32, n = 12922),
         56 heads of 128, sparsity 0.8, with q/k rmsnorm, rope3 and the gate:
         fh3_hip_vsa_attention_qkv_dev -> every VSA kernel
  seqs   attention within packed sequences: fp32 prompts of 37 and 600 tokens
         (64 heads over 8, hd 128), 24 bf16 documents of 17 to 1500 tokens with
         capped scores (40 over 8), 3 fp16 sequences of 1021 to 2047 tokens with
         prefix and distance bias (16 heads of 64), 8192 bf16 tokens (64 over 8):
         fh3_hip_attention_seqs_dev -> k_attn_seqs32, k_attn_seqs16
  cache  the 8-bit cache at 8 key heads of 128: 16 fp32 prompts written and
         read, one bf16 token of 64 sequences likewise, then attention of one
         fp32 token over 300, one bf16 token of 32 sequences of 200 to 8192, one
         fp16 token over 2 x 125000 with distance bias, 2 to 6 fp32 tokens over
         24 x 500 to 5000 with capped scores (16 heads over 4, hd 64), chunks of
         500 bf16 tokens over 2 x 14000 and of 250 fp32 tokens over 2 x 16000:
         fh3_hip_kv_append_dev, _read_dev, _attention_dev -> k_kv_*

  mx     microscaled operands: one FP8 row of 5120 -> 15360 (fp32), 16 of 25600
         -> 5120, 600 of 5120 -> 17408, 8192 FP4 rows of 5120 -> 15360, 3016 FP8
         rows of 7168 -> 5376 (fp32, gated residual), 32768 of 13824 -> 5120
         (gated residual), SwiGLU of 20 x 5120 -> 51200 and 3016 x 5376 ->
         28672, quantisation of 13824 x 5120 fp32 to FP4 and its read-back, of
         37 x 25600 bf16 to FP8, the norm of one fp32 row of 5120 and of 14430
         bf16 rows of 5376, modulated: fh3_hip_mx_* -> k_mx_*; weights rotated

seqs, cache and mx take --only NAME,NAME of their cases.
"""
import argparse
import sys

import numpy as np

from . import fh3 as F

MALL_BYTES = 256 << 20


def gemv(reps):
    for N in (5120, 17408):
        for M in (1, 4, 16):
            K = 5120
            raw = F.synth_q4k_weights(0, 100 + N, N, K, 0.02, 0.0)
            copies = max(2, -(-(MALL_BYTES + (64 << 20)) // raw.nbytes))
            ws = [F.DeviceBuffer.from_array(raw) for _ in range(copies)]
            dx = F.DeviceBuffer.from_array(F.synth_x("normal", 0, 200 + M, M, K))
            dy = F.DeviceBuffer(M * N * 4)
            prep = F.DeviceBuffer(F.prepared_bytes(M, K))
            F.prepare_x_dev(dx, M, K, prep)
            for i in range(reps + 1):
                F.matmul_prepared_dev(ws[i % copies], K, N, prep, dy, M)
            F.synchronize()
            print("gemv M=%d N=%d K=%d: %d launches, %d weight copies" % (M, N, K, reps, copies), flush=True)
            for b in ws + [dx, dy, prep]:
                b.close()


def te(reps):
    for K, N in ((8192, 5120), (25600, 5120)):
        for M in (1, 16):
            raw = F.synth_q4k_weights(0, 100 + N + K, N, K, 0.02, 0.0)
            copies = max(2, -(-(MALL_BYTES + (64 << 20)) // raw.nbytes))
            ws = [F.DeviceBuffer.from_array(raw) for _ in range(copies)]
            dx = F.DeviceBuffer.from_array(F.synth_x("normal", 0, 200 + M, M, K))
            dy = F.DeviceBuffer(M * N * 4)
            prep = F.DeviceBuffer(F.prepared_bytes(M, K))
            F.prepare_x_dev(dx, M, K, prep)
            for i in range(reps + 1):
                F.matmul_prepared_dev(ws[i % copies], K, N, prep, dy, M)
            F.synchronize()
            print("te M=%d N=%d K=%d path %d: %d launches" % (M, N, K, F.matmul_path(M, K), reps), flush=True)
            for b in ws + [dx, dy, prep]:
                b.close()


def _rotated_products(tag, shapes, reps):
    for M, K, N in shapes:
        raw = F.synth_q4k_weights(0, 100 + N + K, N, K, 0.02, 0.0)
        copies = max(2, -(-(MALL_BYTES + (64 << 20)) // raw.nbytes))
        ws = [F.DeviceBuffer.from_array(raw) for _ in range(copies)]
        dx = F.DeviceBuffer.from_array(F.synth_x("normal", 0, 200 + M, M, K))
        dy = F.DeviceBuffer(M * N * 4)
        prep = F.DeviceBuffer(F.prepared_bytes(M, K))
        F.prepare_x_dev(dx, M, K, prep)
        for i in range(reps + 1):
            F.matmul_prepared_dev(ws[i % copies], K, N, prep, dy, M)
        F.synchronize()
        print("%s M=%d N=%d K=%d path %d: %d launches, %d weight copies" % (tag, M, N, K, F.matmul_path(M, K), reps,
                                                                          copies), flush=True)
        for b in ws + [dx, dy, prep]:
            b.close()


def _random_q56(qt, rows, K, seed):
    """Random Q5_K (176 B) or Q6_K (210 B) super-blocks: random quant and
    scale bytes, fp16 block scales (d, and dmin for Q5_K) set to 2^-10."""
    bb = 176 if qt == F.FH3_QUANT_Q5_K else 210
    rng = np.random.default_rng(seed)
    raw = rng.integers(0, 256, size=(rows, K // 256, bb), dtype=np.uint8)
    d = np.frombuffer(np.float16(2.0 ** -10).tobytes(), np.uint8)
    if qt == F.FH3_QUANT_Q5_K:
        raw[:, :, 0:2] = d
        raw[:, :, 2:4] = d
    else:
        raw[:, :, 208:210] = d
    return raw.reshape(-1)


def single(reps):
    M, K, N = 64, 4096, 4096
    raw = F.synth_q4k_weights(0, 100 + N + K, N, K, 0.02, 0.0)
    dw = F.DeviceBuffer.from_array(raw)
    dx = F.DeviceBuffer.from_array(F.synth_x("normal", 0, 200 + M, M, K))
    dy = F.DeviceBuffer(M * N * 4)
    prep = F.DeviceBuffer(F.prepared_bytes(M, K))
    F.prepare_x_dev(dx, M, K, prep)
    for i in range(reps + 1):
        F.matmul_prepared_dev(dw, K, N, prep, dy, M)
    F.synchronize()
    print("single M=%d N=%d K=%d path %d: %d launches, one weight copy" % (M, N, K, F.matmul_path(M, K), reps),
          flush=True)
    for b in (dw, dx, dy, prep):
        b.close()


def q56(reps):
    for qt, K, N in ((F.FH3_QUANT_Q5_K, 5120, 1024), (F.FH3_QUANT_Q6_K, 5120, 1024), (F.FH3_QUANT_Q6_K, 8192, 5120),
                     (F.FH3_QUANT_Q6_K, 25600, 5120)):
        raw = _random_q56(qt, N, K, seed=5)
        copies = max(2, -(-(MALL_BYTES + (64 << 20)) // raw.nbytes))
        ws = [F.DeviceBuffer.from_array(raw) for _ in range(copies)]
        for M in (1, 16, 300):
            dx = F.DeviceBuffer.from_array(F.synth_x("normal", 0, 200 + M, M, K))
            dy = F.DeviceBuffer(M * N * 4)
            prep = F.DeviceBuffer(F.prepared_bytes(M, K))
            F.prepare_x_dev(dx, M, K, prep)
            for i in range(reps + 1):
                F.matmul_prepared_dev(ws[i % copies], K, N, prep, dy, M, qtype=qt)
            F.synchronize()
            print("q56 type %d M=%d N=%d K=%d: %d launches, %d weight copies" % (qt, M, N, K, reps, copies), flush=True)
            for b in (dx, dy, prep):
                b.close()
        for b in ws:
            b.close()


def prompt(reps):
    _rotated_products("prompt", [(M, 5120, N) for N in (5120, 17408) for M in (17, 32, 48, 64)], reps)


def mid(reps):
    _rotated_products("mid", [(M, 5120, N) for N in (5120, 17408) for M in (65, 128, 256)], reps)


def gemm(reps):
    M, K = 8192, 5120
    dx = F.DeviceBuffer.from_array(F.synth_x("outliers", 1, 400 + K, M, K))
    prep = F.DeviceBuffer(F.prepared_bytes(M, K))
    for N in (15360, 5120):
        dw = F.DeviceBuffer.from_array(F.synth_q4k_weights(1, 300 + N + K, N, K, 0.02, 0.0))
        dy = F.DeviceBuffer(M * N * 4)
        for _ in range(reps + 1):
            F.prepare_x_dev(dx, M, K, prep)
            F.matmul_prepared_dev(dw, K, N, prep, dy, M)
        F.synchronize()
        print("gemm M=%d N=%d K=%d: %d launches" % (M, N, K, reps), flush=True)
        dw.close()
        dy.close()


def mlp(reps):
    M = 32768
    for K, N, xkind in ((5120, 13824, "normal"), (13824, 5120, "silu_gated")):
        dx = F.DeviceBuffer.from_array(F.synth_x(xkind, 1, 400 + K, M, K))
        prep = F.DeviceBuffer(F.prepared_bytes(M, K))
        dw = F.DeviceBuffer.from_array(F.synth_q4k_weights(1, 300 + N + K, N, K, 0.02, 2.0))
        dy = F.DeviceBuffer(M * N * 4)
        for _ in range(reps + 1):
            F.prepare_x_dev(dx, M, K, prep)
            F.matmul_prepared_dev(dw, K, N, prep, dy, M)
        F.synchronize()
        print("mlp M=%d N=%d K=%d: %d launches" % (M, N, K, reps), flush=True)
        for b in (dx, prep, dw, dy):
            b.close()


def copy(reps):
    n = 256 << 20
    a, b = F.DeviceBuffer(n), F.DeviceBuffer(n)
    a.fill(1)
    for _ in range(reps + 1):
        F._check(F.lib().fh3_hip_memcpy_dtod(b.ptr, a.ptr, n), "fh3_hip_memcpy_dtod")
    F.synchronize()
    print("copy %d bytes: %d launches" % (n, reps), flush=True)


def attn(reps, n=16384, heads=40, hd=128, rot=96):
    inner = heads * hd
    qkv = F.DeviceBuffer.from_array(F.synth_x("normal", 2, 500, n, 3 * inner))
    w = F.DeviceBuffer.from_array(np.ones(hd, np.float32))
    ang = np.outer(np.arange(n, dtype=np.float64), 1e-2 * np.arange(1, rot // 2 + 1))
    ang = np.concatenate([ang, ang], axis=1)
    cs = F.DeviceBuffer.from_array(np.cos(ang).astype(np.float32))
    sn = F.DeviceBuffer.from_array(np.sin(ang).astype(np.float32))
    o = F.DeviceBuffer(n * inner * 4)
    for _ in range(reps + 1):
        F.attention_qkv_dev(qkv, n, heads, hd, o, w, w, 1e-5, cs, sn, rot)
    F.synchronize()
    print("attn n=%d heads=%d hd=%d: %d launches" % (n, heads, hd, reps), flush=True)
    for b in (qkv, w, cs, sn, o):
        b.close()


def vsa(reps, heads=56, hd=128, rot=96):
    n_text, n_audio, grid = 6, 244, (22, 18, 32)
    n = n_text + n_audio + grid[0] * grid[1] * grid[2]
    inner = heads * hd
    qkv = F.DeviceBuffer.from_array(F.synth_x("normal", 4, 700, n, 3 * inner))
    gate = F.DeviceBuffer.from_array(F.synth_x("normal", 4, 701, n, inner))
    w = F.DeviceBuffer.from_array(np.ones(hd, np.float32))
    ang = np.outer(np.arange(n, dtype=np.float64), 1e-2 * np.arange(1, rot // 2 + 1))
    ang = np.concatenate([ang, ang], axis=1)
    cs = F.DeviceBuffer.from_array(np.cos(ang).astype(np.float32))
    sn = F.DeviceBuffer.from_array(np.sin(ang).astype(np.float32))
    o = F.DeviceBuffer(n * inner * 4)
    seq = F.seq_of(n, n_text, n_audio, grid=grid)
    for _ in range(reps + 1):
        F.vsa_attention_qkv_dev(qkv, gate, o, seq, heads, hd, 0.8, 64, w, w, 1e-5, cs, sn, rot)
    F.synchronize()
    print("vsa n=%d heads=%d hd=%d: %d launches" % (n, heads, hd, reps), flush=True)
    for b in (qkv, gate, w, cs, sn, o):
        b.close()


_TYPES = {"F32": F.FH3_QUANT_F32, "F16": F.FH3_QUANT_F16, "BF16": F.FH3_QUANT_BF16}


def _typed(rng, n, width, t, scale=1.0):
    x = rng.standard_normal((n, width), dtype=np.float32) * np.float32(scale)
    x = x if t == "F32" else x.astype(np.float16) if t == "F16" else (x.view(np.uint32) >> 16).astype(np.uint16)
    return F.DeviceBuffer.from_array(x)


def _spread(rng, n, lo, hi):
    return [int(x) for x in np.exp(rng.uniform(np.log(lo), np.log(hi), n)).round()]


def _first(lens):
    return F.DeviceBuffer.from_array(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))


def _slopes(heads):
    return F.DeviceBuffer.from_array((2.0 ** (-8.0 * (np.arange(heads) + 1) / heads)).astype(np.float32))


def seqs(reps, only=None):
    rng = np.random.default_rng(3)
    cases = [("prompt_37", "F32", 64, 8, 128, [37], 0.0, False, 0.0), ("prompt_600", "F32", 64, 8, 128, [600], 0.0, False, 0.0),
             ("documents", "BF16", 40, 8, 128, _spread(rng, 24, 17, 1500), 50.0, False, 0.0),
             ("prefix", "F16", 16, 16, 64, _spread(rng, 3, 1021, 2047), 0.0, True, 0.25),
             ("long", "BF16", 64, 8, 128, [8192], 0.0, False, 0.0)]
    for name, t, heads, kv, hd, lens, cap, bias, prefix in cases:
        if only and name not in only:
            continue
        n = sum(lens)
        q, k, v = (_typed(rng, n, w * hd, t, s) for w, s in ((heads, 1.5), (kv, 1.0), (kv, 1.0)))
        o, first = F.DeviceBuffer(q.nbytes), _first(lens)
        pre = F.DeviceBuffer.from_array(np.asarray([int(x * prefix) for x in lens], np.int32)) if prefix else None
        slopes = _slopes(heads) if bias else None
        cfg = F.attn_cfg(heads, kv, hd, _TYPES[t], softcap=cap, d_slopes=slopes)
        for _ in range(reps + 1):
            F.attention_seqs_dev(cfg, q, k, v, o, n, len(lens), first, pre)
        F.synchronize()
        print("seqs %s: %s, %d tokens, %d launches" % (name, t, n, reps), flush=True)
        for b in (q, k, v, o, first, pre, slopes):
            if b is not None:
                b.close()


def cache(reps, only=None):
    rng = np.random.default_rng(4)
    cases = [("fill", "F32", 0, 8, 128, [0] * 16, _spread(rng, 16, 100, 600), 0.0, False),
             ("append", "BF16", 0, 8, 128, _spread(rng, 64, 100, 4000), [1] * 64, 0.0, False),
             ("token", "F32", 64, 8, 128, [299], [1], 0.0, False),
             ("batch", "BF16", 64, 8, 128, _spread(rng, 32, 200, 8192), [1] * 32, 0.0, False),
             ("far", "F16", 40, 8, 128, [125000] * 2, [1] * 2, 0.0, True),
             ("few", "F32", 16, 4, 64, _spread(rng, 24, 500, 5000), [2 + i % 5 for i in range(24)], 30.0, False),
             ("chunk", "BF16", 64, 8, 128, [13500] * 2, [500] * 2, 0.0, False),
             ("chunk_fp32", "F32", 64, 8, 128, [15750] * 2, [250] * 2, 0.0, False)]
    for name, t, heads, kv, hd, held, new, cap, bias in cases:
        if only and name not in only:
            continue
        lens = [a + b for a, b in zip(held, new)]
        need = [-(-x // F.KV_PAGE) for x in lens]
        pages, n, n_seq = sum(need), sum(new), len(new)
        raw = np.empty(F.kv_pool_bytes(kv, hd, pages), np.uint8)
        split = raw.nbytes - pages * kv * 2 * 4
        raw[:split] = rng.integers(1, 256, split, dtype=np.uint8)
        raw[split:] = np.full(pages * kv * 2, 2.0 ** -6, np.float32).view(np.uint8)
        table, order = np.full((n_seq, max(need)), -1, np.int32), rng.permutation(pages)
        for i, (a, b) in enumerate(zip(np.cumsum([0] + need), need)):
            table[i, :b] = order[a:a + b]
        pool, table, length = (F.DeviceBuffer.from_array(x) for x in (raw, table, np.asarray(lens, np.int32)))
        first = _first(new)
        c, used = F.kv_cache(kv, hd, pages, max(need), pool, table, length), [pool, table, length, first]
        if heads:
            q, slopes = _typed(rng, n, heads * hd, t, 0.3), _slopes(heads) if bias else None
            o = F.DeviceBuffer(q.nbytes)
            cfg = F.attn_cfg(heads, kv, hd, _TYPES[t], softcap=cap, d_slopes=slopes)
            size = F.kv_attention_workspace_bytes(cfg, c, n, n_seq)
            ws = F.DeviceBuffer(max(1, size))
            used += [q, o, ws] + ([slopes] if bias else [])
            for _ in range(reps + 1):
                F.kv_attention_dev(cfg, c, q, o, n, n_seq, ws, size, first)
        else:
            back = [x - (x - a) // F.KV_PAGE * F.KV_PAGE for x, a in zip(lens, new)]   # all of the touched pages
            k, v, ko, vo = (_typed(rng, m, kv * hd, t) for m in (n, n, sum(back), sum(back)))
            bf = _first(back)
            used += [k, v, ko, vo, bf]
            for _ in range(reps + 1):
                F.kv_append_dev(c, _TYPES[t], k, v, n, n_seq, first)
                F.kv_read_dev(c, _TYPES[t], ko, vo, sum(back), n_seq, bf)
        F.synchronize()
        print("cache %s: %s, %d tokens held, %d new, %d launches" % (name, t, sum(lens), n, reps), flush=True)
        for b in used:
            b.close()


def _mx_rows(rng, fmt, rows, n):
    """Random codes (FP8: without NaN) and scales of 2^-3 to 2^3."""
    codes, scales = (np.empty(b, np.uint8) for b in F.mx_bytes(fmt, rows, n))
    codes[:] = rng.integers(0, 256, codes.size, dtype=np.uint8) & (0xFF if fmt == F.FH3_MX_FP4 else 0xF7)
    scales[:] = rng.integers(124, 131, scales.size, dtype=np.uint8)
    c, s = F.DeviceBuffer.from_array(codes), F.DeviceBuffer.from_array(scales)
    return F.mx(fmt, rows, n, c, s), [c, s]


def mx(reps, only=None):
    rng = np.random.default_rng(5)
    fp4, fp8 = F.FH3_MX_FP4, F.FH3_MX_FP8
    products = [("token", fp8, 1, 5120, 15360, "F32", False), ("tokens", fp8, 16, 25600, 5120, "BF16", False),
                ("prompt", fp8, 600, 5120, 17408, "BF16", False), ("clip", fp4, 8192, 5120, 15360, "BF16", False),
                ("out", fp8, 3016, 7168, 5376, "F32", True), ("long", fp8, 32768, 13824, 5120, "BF16", True),
                ("prompt_swiglu", fp8, 20, 5120, 51200, None, False), ("clip_swiglu", fp8, 3016, 5376, 28672, None, False)]
    for name, fmt, rows, n, out, t, gated in products:
        if only and name not in only:
            continue
        used = []
        x, b = _mx_rows(rng, fmt, rows, n)
        used += b
        ws = []
        for _ in range(max(1, min(8, MALL_BYTES // (out * n // 2))) + 1 if rows <= 64 else 1):
            w, b = _mx_rows(rng, fp4, out, n)
            ws.append(w)
            used += b
        size = F.mx_matmul_workspace_bytes(ws[0], x, t is None)
        work = F.DeviceBuffer(max(1, size))
        used.append(work)
        if t is None:
            y, b = _mx_rows(rng, fp8, rows, out // 2)
            used += b
        else:
            y = F.DeviceBuffer(rows * out * (4 if t == "F32" else 2))
            used.append(y)
        res, gate = None, None
        if gated:
            res, gate = _typed(rng, rows, out, t), _typed(rng, rows, out, "F32")
            used += [res, gate]
        for i in range(reps + 1):
            if t is None:
                F.mx_matmul_swiglu_dev(ws[i % len(ws)], x, y, work, size)
            else:
                F.mx_matmul_dev(ws[i % len(ws)], x, _TYPES[t], y, work, size, d_gate=gate, d_res=res)
        F.synchronize()
        print("mx %s: %d x %d -> %d, %d launches" % (name, rows, n, out, reps), flush=True)
        for b in used:
            b.close()
    for name, fmt, rows, n, t in (("weights", fp4, 13824, 5120, "F32"), ("rows", fp8, 37, 25600, "BF16")):
        if only and name not in only:
            continue
        x, back = _typed(rng, rows, n, t), F.DeviceBuffer(rows * n * 2)
        y, used = _mx_rows(rng, fmt, rows, n)
        for _ in range(reps + 1):
            F.mx_quantize_dev(_TYPES[t], x, y)
            F.mx_dequant_dev(y, F.FH3_QUANT_BF16, back)
        F.synchronize()
        print("mx %s: %d x %d, %d launches" % (name, rows, n, reps), flush=True)
        for b in [x, back] + used:
            b.close()
    for name, rows, n, t, mod in (("token_norm", 1, 5120, "F32", False), ("clip_norm", 14430, 5376, "BF16", True)):
        if only and name not in only:
            continue
        x, add, w = _typed(rng, rows, n, t), _typed(rng, rows, n, t), _typed(rng, 1, n, "F32")
        shift, scale = (_typed(rng, rows, n, "F32") for _ in range(2)) if mod else (None, None)
        y, used = _mx_rows(rng, fp8, rows, n)
        total = F.DeviceBuffer(x.nbytes)
        for _ in range(reps + 1):
            F.mx_norm_dev(_TYPES[t], x, w, 1e-6, y, d_add=add, d_sum=total, d_shift=shift, d_scale=scale)
        F.synchronize()
        print("mx %s: %d x %d, %d launches" % (name, rows, n, reps), flush=True)
        for b in [x, add, w, total] + used + ([shift, scale] if mod else []):
            b.close()


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("workload", choices=("gemv", "te", "prompt", "mid", "single", "q56", "gemm", "mlp", "copy", "attn", "vsa",
                                         "seqs", "cache", "mx", "all"))
    ap.add_argument("--reps", type=int, default=20)
    ap.add_argument("--only", help="seqs, cache, mx: these cases")
    args = ap.parse_args(argv)
    F.init(0)
    if args.workload in ("seqs", "cache", "mx"):
        globals()[args.workload](args.reps, args.only.split(",") if args.only else None)
        return 0
    for name in (("gemv", "gemm", "copy") if args.workload == "all" else (args.workload,)):
        globals()[name](args.reps)
    return 0


if __name__ == "__main__":
    sys.exit(main())
