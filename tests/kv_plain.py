"""The KV cache's formats and the attentions over it, restated plainly for the tests: numpy f32 for the quantisers (every
rounding is part of their definition), torch f64 on the host for the attention, a row and a head at a time."""
from __future__ import annotations

import math

import numpy as np
import torch

BLOCK = 32


def quantise(x: np.ndarray, kind: str) -> tuple[np.ndarray, np.ndarray]:
    """f32 [..., d] → (quants as signed integers [..., d], f16 scales [..., d / 32])"""
    xb = x.astype(np.float32).reshape(*x.shape[:-1], -1, BLOCK)
    bad = ~np.isfinite(xb).all(-1)
    xb = np.where(bad[..., None], np.float32(0), xb)
    if kind == "q8_0":
        step = np.abs(xb).max(-1) / np.float32(127)
    else:
        first = np.abs(xb).argmax(-1)  # numpy's argmax keeps the first
        step = np.take_along_axis(xb, first[..., None], -1)[..., 0] / np.float32(-8)
    with np.errstate(over="ignore", divide="ignore", invalid="ignore"):
        scale = step.astype(np.float16)
        bad |= ~np.isfinite(scale)
        live = (scale != 0) & ~bad
        y = np.where(live[..., None], xb * (np.float32(1) / step)[..., None], np.float32(0)).astype(np.float32)
    if kind == "q8_0":
        a = np.abs(y)
        q = np.copysign(np.floor(a) + ((a - np.floor(a)) >= 0.5), y)
    else:
        q = np.minimum(np.floor(y + np.float32(8.5)), 15) - 8
    scale = np.where(bad, np.float16(np.nan), scale)
    return q.astype(np.int32).reshape(x.shape), scale


def held(x: np.ndarray, kind: str) -> np.ndarray:
    """the values that the cache stands for, f32"""
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float32)
    q, s = quantise(x, kind)
    return (q.reshape(*s.shape, BLOCK).astype(np.float32) * s.astype(np.float32)[..., None]).reshape(x.shape)


def packed(q: np.ndarray, kind: str) -> np.ndarray:
    """signed quants → the cache's bytes"""
    if kind == "q8_0":
        return q.astype(np.int8)
    b = (q + 8).astype(np.uint8).reshape(*q.shape[:-1], -1, 2, 16)
    return (b[..., 0, :] | (b[..., 1, :] << 4)).reshape(*q.shape[:-1], -1)


def row_of(p: int, n_rows: int, sinks: int, ring: bool) -> int:
    return sinks + (p - sinks) % (n_rows - sinks) if ring and p >= sinks else p


def depths(parent) -> list[int]:
    d = []
    for p in parent:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def sees(pos: int, t: int, j: int, window: int, sinks: int, parent=None) -> bool:
    """whether row t of a call at pos sees the key that was written as position j"""
    mine, theirs = pos + t, j
    if parent is not None:
        d = depths(parent)
        mine = pos + d[t]
        if j >= pos:
            i = t
            while i > j - pos:
                i = parent[i]
            if i != j - pos:
                return False
            theirs = pos + d[j - pos]
    elif j > mine:
        return False
    return window == 0 or theirs > mine - window or theirs < sinks


def mask_of(pos: int, T: int, window: int, sinks: int, parent=None) -> torch.Tensor:
    """sees() of every row and position at once"""
    where = torch.arange(pos + T)
    if parent is None:
        mine = where[pos:]
        seen = where[None] <= mine[:, None]
    else:
        d = torch.tensor(depths(parent))
        where = torch.cat([where[:pos], pos + d])
        mine = pos + d
        seen = torch.zeros(T, pos + T, dtype=torch.bool)
        for t, p in enumerate(parent):
            seen[t, :pos] = True
            if p >= 0:
                seen[t, pos:] = seen[p, pos:]
            seen[t, pos + t] = True
    if window:
        seen &= (where[None] > mine[:, None] - window) | (where[None] < sinks)
    return seen


def attend(q, keys, values, pos: int, scale: float, window: int = 0, sinks: int = 0, parent=None):
    """q [T][n_head][d]; keys, values [n_kv][positions][d] in order of position (the call's own rows last), f64 → [T][n_head][d]"""
    T, H, d = q.shape
    G = H // keys.shape[0]
    n = pos + T
    mask = mask_of(pos, T, window, sinks, parent)
    out = torch.zeros(T, H, d, dtype=torch.float64)
    for h in range(H):
        k, v = keys[h // G, :n], values[h // G, :n]
        bad = ~torch.isfinite(v)
        s = torch.where(mask, (q[:, h] @ k.T) * scale, -math.inf)
        p = torch.exp(s - s.max(-1, keepdim=True).values)
        p = torch.where(mask, p, 0.0)  # (a row that sees nothing)
        o = p @ torch.where(bad, 0.0, v) / p.sum(-1, keepdim=True)
        o[(mask.double() @ bad.double()) > 0] = math.nan
        out[:, h] = torch.where(mask.any(-1, keepdim=True), o, 0.0)
    return out
