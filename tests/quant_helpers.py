"""Caches and matrices in codes, restated with numpy in 64 bits, and the errors that arithmetic allows the kernels."""
import numpy as np
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def to_bf16(x):
    """fp64 -> the nearest number of 8 significant bits, ties to even (normal range)."""
    m, e = np.frexp(np.asarray(x, np.float64))
    return np.ldexp(np.rint(m * 256.0), e - 8)


def quantise(x, bits):
    """Rows x (fp64, finite) -> (codes int64, scale, zero), by the definition."""
    q = 2 ** bits - 1
    low, high = np.minimum(x.min(-1, keepdims=True), 0.0), np.maximum(x.max(-1, keepdims=True), 0.0)
    scale = to_bf16((high - low).astype(np.float32).astype(np.float64) / q)
    div = np.where(scale > 0, scale, 1.0)
    zero = np.clip(np.rint(-low / div), 0, q)
    code = np.clip(np.rint(x / div) + zero, 0, q)
    return np.where(scale > 0, code, 0).astype(np.int64), scale, np.where(scale > 0, zero, 0).astype(np.int64)


def pack(codes, bits):
    codes = codes.astype(np.uint8)
    return codes if bits == 8 else codes[..., 0::2] | (codes[..., 1::2] << 4)


def unpack(codes, bits):
    return codes.astype(np.int64) if bits == 8 else np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1).astype(np.int64)


def parameters(scale, zero):
    """[..., 2] int16 from [..., 1]."""
    pattern = (scale.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
    return np.concatenate([pattern.view(np.int16), zero.astype(np.int16)], -1)


def scale_zero(params):
    scale = (params[..., 0].astype(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return scale, params[..., 1].astype(np.float64)


def values(codes, params, bits):
    scale, zero = scale_zero(params)
    return scale[..., None] * (unpack(codes, bits) - zero[..., None])


def int8_rows(x):
    scale = to_bf16(np.abs(x).max(-1, keepdims=True) / 127)
    return np.where(scale > 0, np.clip(np.rint(x / np.where(scale > 0, scale, 1.0)), -127, 127), 0.0), scale[..., 0]


def host(t):
    return t.detach().cpu().numpy()


def wide(t):
    return t.detach().double().cpu().numpy()


def fill(cache, layer, seed, scale=1.0):
    """Random rows, quantised here, in every slot of a layer; some features larger throughout, as keys have them."""
    rng = np.random.default_rng(seed)
    l = cache.layers[layer]
    B, heads, cap, _ = l.k_codes.shape
    big = 1.0 + 3.0 * (rng.random(cache.head_dim) < 0.1)
    for codes, params in ((l.k_codes, l.k_params), (l.v_codes, l.v_params)):
        c, s, z = quantise(rng.standard_normal((B, heads, cap, cache.head_dim)) * big * scale, cache.bits)
        codes.copy_(torch.from_numpy(pack(c, cache.bits)))
        params.copy_(torch.from_numpy(parameters(s, z)))


def attention(cache, layer, q, row_start, kv_begin, base_len, mode, tree_mask, scale, weight_step, exp_step=2.0 ** -20):
    """(out, bound): attention in 64 bits over the values that the codes stand for, [tokens, heads * dim], and how far a kernel may be off
    whose softmax weights are rounded by at most weight_step (relative) beside what fp32 sums of scores cost; a row that sees nothing is 0.

    Weights in fp16 have a smallest step besides, which counts where a feature's large weights all meet values of 0.  In the kernel for few rows a weight
    is p s / r 2^14, s the value's scale, r the largest scale R of the keys; the largest p is at least 1 and the sum l that the result is divided
    by too.  Half of fp16's smallest step is 2^-25, so a key adds at most 2^-25 2^-14 r (code - zero) / l <= 2^-39 R (2^bits - 1).

    The kernel for many rows rounds keys and values, scales and all, to fp16: 2^-12 of each, so a score is off by 2^-12 sum |q k| scale.  Its
    weights are 2^7 p, of values s / r 2^6 (code - zero) or more: a key adds 2^-25 2^-7 R (2^bits - 1), a value's own smallest step 2^-31 R.

    The kernel for few rows sums W code and W zero apart, in fp32, and takes one from the other, which shows where values cancel or are 0.  A
    product of 16 keys adds to a sum of at most (2^bits - 1) R times the weights' share; a tensor core's addition may cut 2^-23 of that, the sum
    of W zero, an addition for each of a lane's keys, too, and so may the difference.  A warp, one of eight, has n / 128 such products, two
    more at the ends: (n / 128 + 2) 2^-22 (2^bits - 1) R in all."""
    l = cache.layers[layer]
    B, heads, cap, _ = l.k_codes.shape
    hd = cache.head_dim
    q = np.asarray(q, np.float64)
    m = q.shape[0]
    nh = q.shape[1] // hd
    k, v = values(host(l.k_codes), host(l.k_params), cache.bits), values(host(l.v_codes), host(l.v_params), cache.bits)
    ks = scale_zero(host(l.k_params))[0]
    vs = np.nan_to_num(scale_zero(host(l.v_params))[0])
    top = 2 ** cache.bits - 1
    out, bound = np.zeros((m, nh, hd)), np.zeros((m, nh, hd))
    for b in range(B):
        s, e, first, base = row_start[b], row_start[b + 1], kv_begin[b], base_len[b]
        n = e - s
        for i in range(n):
            new = np.arange(n) <= i if mode == 0 else np.array([(int(tree_mask[s + i, j >> 5]) >> (j & 31)) & 1 for j in range(n)], bool)
            seen = first + np.flatnonzero(np.concatenate([np.ones(base, bool), new]))
            if seen.size == 0:
                continue
            for h in range(nh):
                g = h // (nh // heads)
                x = q[s + i, h * hd : (h + 1) * hd]
                sc = k[b, g, seen] @ x * scale
                p = np.exp(sc - sc.max())
                p /= p.sum()
                out[s + i, h] = p @ v[b, g, seen]
                # Sums in fp32 of hd products of a query and a code (up to `top`) and of zero * sum q: hd + 4 roundings of 2^-23 (the tensor
                # core cuts) of their absolute sum; one 2^-22 for the scaling and e^x's argument, relative to the score.
                err = (hd + 4) * 2.0 ** -23 * np.abs(x).sum() * 2 * top * ks[b, g, seen].max() * abs(scale) + 2.0 ** -22 * np.abs(sc).max()
                if weight_step > 2.0 ** -12:
                    err += 2.0 ** -12 * (np.abs(k[b, g, seen]) @ np.abs(x)).max() * abs(scale)
                weight = weight_step + exp_step + 2 * err + seen.size * 2.0 ** -23
                bound[s + i, h] = weight * (p @ np.abs(v[b, g, seen])) + weight * np.abs(out[s + i, h])
                if weight_step > 2.0 ** -12:
                    bound[s + i, h] += (seen.size * 2.0 ** -32 + (seen.size / 128 + 2) * 2.0 ** -22) * vs[b, g, seen].max() * top
    return out.reshape(m, -1), bound.reshape(m, -1)


def trees(counts, seed, words=None):
    """Packed draft trees: [tokens, words] int32, bit j of a token's row set for itself and its ancestors."""
    rng = np.random.default_rng(seed)
    words = words or max(1, (max(counts) + 31) // 32)
    mask = np.zeros((sum(counts), words), np.uint32)
    t = 0
    for n in counts:
        depth = []
        for i in range(n):
            parents = [j for j in range(i) if depth[j] < 7]
            if parents and rng.random() < 0.9:
                j = int(rng.choice(parents))
                mask[t + i] = mask[t + j]
                depth.append(depth[j] + 1)
            else:
                depth.append(0)
            mask[t + i, i >> 5] |= np.uint32(1 << (i & 31))
        t += n
    return mask.view(np.int32)


def starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")
