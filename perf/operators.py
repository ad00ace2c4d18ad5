"""Operators around the splash attention kernels, as measurable cases: each with a plain form in elementary torch
operations and with the calls that a user makes of the library (`own`).

  rotary   rotary positions with one or several axes (time, height, width) on q and k, forward and backward
  write    new keys and values into a paged cache, as 16-bit or as 8-bit numbers with a power-of-two scale per (token, head)
  read     the keys and values of a batch of sequences out of such a cache
  attend   attention of one token, a run of tokens or a tree of drafted tokens per sequence over the cache
  sinks    sliding-window attention with a few first tokens that stay visible, inference and training

Sizes common to the cases: batch, heads, kv_heads, n (new tokens or positions per sequence), head_dim, dtype (of q, k, v).  A cache has
pages of `page` tokens, [pages, kv_heads, page, head_dim]; the sequences of a batch own random pages of it, and their lengths are
min_len..max_len (drawn from the seed of the inputs).
"""

import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "pallas-mosaic-gpu_b200")
DEVICE = "cuda"
MIN_EXPONENT, MAX_EXPONENT = -64, 120


def _library():
  if PACKAGE not in sys.path:
    sys.path.insert(0, PACKAGE)
  import splash_attention_mgpu
  return splash_attention_mgpu


def _case(**kw):
  c = dict(op="attend", batch=1, heads=8, kv_heads=8, n=1, head_dim=128, dtype="bf16", page=64, quantized=False,
           min_len=0, max_len=0, ragged_new=False, tree=False, window=-1, sinks=0, cap=0.0, lse=False,
           train=False, axes=1, adjacent=False, fused_qkv=False, kv_len=0)
  c.update(kw)
  return c


def listed():
  return [
      # One decoding step of a batch: q and k are views of one projection's output.
      _case(name="rotary_token", op="rotary", batch=32, heads=32, kv_heads=8, n=1, fused_qkv=True),
      # Training on video and text, positions of three axes, an odd length.
      _case(name="rotary_video_train", op="rotary", batch=2, heads=32, kv_heads=8, n=8191, axes=3, train=True),
      # The new token of every sequence of a batch goes into the 8-bit cache.
      _case(name="write_token_8bit", op="write", batch=64, kv_heads=8, n=1, quantized=True, min_len=500, max_len=2000,
            fused_qkv=True),
      # Prompts of different lengths go into the 8-bit cache.
      _case(name="write_prompt_8bit", op="write", batch=4, kv_heads=8, n=8192, quantized=True, min_len=0, max_len=4000,
            ragged_new=True),
      # The cached keys of a batch are laid out for the prefill kernels.
      _case(name="read_prompt_8bit", op="read", batch=4, kv_heads=8, quantized=True, min_len=3000, max_len=16384, page=16),
      # A small model answers a few users: one token each against short contexts.
      _case(name="token_small_d64", batch=4, heads=16, kv_heads=4, head_dim=64, dtype="f16", min_len=1, max_len=700, page=16),
      # The ordinary decoding step of a batch with long contexts, grouped heads.
      _case(name="token_long", batch=16, heads=32, kv_heads=8, min_len=4000, max_len=32768, lse=True),
      # The same from the 8-bit cache, more heads to a group.
      _case(name="token_long_8bit", batch=32, heads=64, kv_heads=8, min_len=2000, max_len=32768, quantized=True),
      # Verification of a tree of drafted tokens.
      _case(name="tree_48", batch=8, heads=32, kv_heads=8, n=48, tree=True, min_len=1000, max_len=8192),
      # Streaming chat: windowed layers with sinks, soft-capped logits, a run of four drafted tokens, 8-bit cache.
      _case(name="window_sinks_run_8bit", batch=64, heads=32, kv_heads=8, n=4, min_len=300, max_len=32768, window=4095,
            sinks=4, cap=50.0, quantized=True, ragged_new=True),
      # Training step with a sliding window and sinks, grouped heads.
      _case(name="sinks_train", op="sinks", batch=1, heads=8, kv_heads=2, n=8192, window=1023, sinks=4, train=True),
      # A chunk of a prompt against what came before it.
      _case(name="sinks_prefill_d64", op="sinks", batch=1, heads=32, kv_heads=8, n=1024, kv_len=16384, head_dim=64, dtype="f16",
            window=4095, sinks=16),
  ]


def _spread(rng, lo, hi):
  """Whole number in [lo, hi], spread over its logarithm."""
  return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
  op = rng.choice(("rotary", "write", "read", "attend", "attend", "attend", "sinks"))
  kv_heads = rng.choice((1, 2, 4, 8))
  group = rng.choice((1, 2, 4, 8))
  common = dict(op=op, kv_heads=kv_heads, heads=kv_heads * group, head_dim=rng.choice((64, 128)),
                dtype=rng.choice(("bf16", "f16")), page=rng.choice((16, 32, 64, 128)))
  if op == "rotary":
    c = _case(**common, batch=rng.choice((1, 2, 4, 32)), n=_spread(rng, 1, 8192), axes=rng.choice((1, 2, 3)),
              train=rng.random() < 0.5, adjacent=rng.random() < 0.3, fused_qkv=rng.random() < 0.5)
    while c["batch"] * c["heads"] * c["n"] * c["head_dim"] > 2 * 32 * 8192 * 128:
      c["n"] = (c["n"] + 1) // 2
  elif op in ("write", "read"):
    c = _case(**common, batch=_spread(rng, 1, 64), n=_spread(rng, 1, 8192), quantized=rng.random() < 0.6,
              max_len=_spread(rng, 16, 16384), ragged_new=rng.random() < 0.5, fused_qkv=rng.random() < 0.5)
    c["min_len"] = rng.randint(0, c["max_len"])
    while c["batch"] * max(c["n"], c["max_len"]) > 4 * 16384:
      c["batch"] = (c["batch"] + 1) // 2
  elif op == "attend":
    kind = rng.choice(("token", "token", "run", "tree"))
    n = 1 if kind == "token" else _spread(rng, 2, 16) if kind == "run" else rng.randint(5, 64)
    c = _case(**common, batch=_spread(rng, 1, 64), n=n, tree=kind == "tree", ragged_new=n > 1 and rng.random() < 0.5,
              quantized=rng.random() < 0.5, max_len=_spread(rng, 64, 32768), lse=rng.random() < 0.3,
              cap=rng.choice((0.0, 0.0, 30.0)))
    c["min_len"] = rng.randint(0, c["max_len"])
    if rng.random() < 0.4:
      c["window"], c["sinks"] = _spread(rng, 64, 8192), rng.choice((0, 4, 64))
    while c["batch"] * c["max_len"] * (c["kv_heads"] + c["heads"] * n / 32) * c["head_dim"] > 16 * 32768 * 9 * 128:
      if c["batch"] > 1:
        c["batch"] = (c["batch"] + 1) // 2
      else:
        c["max_len"], c["min_len"] = c["max_len"] // 2, c["min_len"] // 2
  else:
    c = _case(**common, batch=rng.choice((1, 1, 2)), n=128 * _spread(rng, 1, 64), window=_spread(rng, 32, 4096),
              sinks=rng.choice((1, 4, 16, 200)), cap=rng.choice((0.0, 0.0, 30.0)), train=rng.random() < 0.6)
    if not c["train"] and rng.random() < 0.5:
      c["kv_len"] = c["n"] + 128 * _spread(rng, 1, 64)
    while c["batch"] * c["heads"] * c["n"] * max(c["n"], c["kv_len"]) > 8 * 8192 * 8192:
      if c["heads"] > c["kv_heads"]:
        c["heads"] //= 2
      elif c["kv_heads"] > 1:
        c["kv_heads"] //= 2
        c["heads"] //= 2
      elif c["batch"] > 1:
        c["batch"] //= 2
      else:
        c["n"] = 128 * max(1, c["n"] // 256)
  return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _dtype(c):
  return torch.bfloat16 if c["dtype"] == "bf16" else torch.float16


def _generator(seed):
  return torch.Generator(device=DEVICE).manual_seed(seed)


def _lengths(c, seed):
  """Tokens in the cache per sequence before the new ones, and new tokens per sequence."""
  rng = np.random.default_rng(seed)
  before = rng.integers(c["min_len"], c["max_len"] + 1, c["batch"])
  new = rng.integers(0, c["n"] + 1, c["batch"]) if c["ragged_new"] else np.full(c["batch"], c["n"])
  return before.astype(np.int64), new.astype(np.int64)


def _heads_of(c, g, heads):
  """[batch, heads, n, head_dim] normal numbers: contiguous, or a view of the output [batch, n, all heads, head_dim] of a projection."""
  shape = (c["batch"], c["n"], heads, c["head_dim"]) if c["fused_qkv"] else (c["batch"], heads, c["n"], c["head_dim"])
  x = torch.randn(shape, generator=g, device=DEVICE).to(_dtype(c))
  return x.transpose(1, 2) if c["fused_qkv"] else x


def _sections(c):
  pairs = c["head_dim"] // 2
  if c["axes"] == 1:
    return (pairs,)
  if c["axes"] == 2:
    return (pairs // 2, pairs // 2)
  return (pairs // 4, 3 * pairs // 8, 3 * pairs // 8)


def _positions(c, seed):
  """[batch, axes, n] whole positions (one axis: [batch, n]): text that goes on from a far position, video as time, height, width."""
  rng = np.random.default_rng(seed)
  start = rng.integers(0, 100000, c["batch"])
  i = np.arange(c["n"])
  if c["axes"] == 1:
    p = start[:, None] + i[None]
  else:
    grid = (i // 1024, i // 32 % 32, i % 32)
    p = start[:, None, None] + np.stack([grid[3 - c["axes"] + a] for a in range(c["axes"])])[None]
  return torch.from_numpy(p.astype(np.int32)).to(DEVICE)


def _parents(c, seed):
  """[batch, n] a random tree per sequence: node i hangs on one of the nodes before it, or (-1) on the last cached token."""
  rng = np.random.default_rng(seed)
  p = np.full((c["batch"], c["n"]), -1, np.int32)
  for i in range(1, c["n"]):
    p[:, i] = np.where(rng.random(c["batch"]) < 0.15, -1, rng.integers(max(0, i - 8), i, c["batch"]))
  return p


def _table(c, tokens, g):
  """Pages of the sequences: [batch, pages per sequence] random, distinct pages of a cache with a few pages to spare."""
  per = -(-max(1, tokens) // c["page"])
  perm = torch.randperm(c["batch"] * per + 3, generator=g, device=DEVICE)[:c["batch"] * per]
  return perm.view(c["batch"], per).to(torch.int32), c["batch"] * per + 3


def _cache(c, pages, g, filled):
  """Buffers of a cache.  `filled`: with keys and values in every slot (8 bit: codes and exponents as they come from normal numbers)."""
  shape = (pages, c["kv_heads"], c["page"], c["head_dim"])
  if not c["quantized"]:
    make = (lambda: torch.randn(shape, generator=g, device=DEVICE, dtype=_dtype(c))) if filled else (
        lambda: torch.zeros(shape, device=DEVICE, dtype=_dtype(c)))
    return {"k": make(), "v": make(), "k_exponent": None, "v_exponent": None}
  if not filled:
    zeros = lambda: torch.zeros(shape, device=DEVICE, dtype=torch.uint8).view(torch.float8_e4m3fn)
    exps = lambda: torch.zeros(shape[:3], device=DEVICE, dtype=torch.int8)
    return {"k": zeros(), "v": zeros(), "k_exponent": exps(), "v_exponent": exps()}
  k, ke = _quantize(torch.randn(shape, generator=g, device=DEVICE, dtype=_dtype(c)))
  v, ve = _quantize(torch.randn(shape, generator=g, device=DEVICE, dtype=_dtype(c)))
  return {"k": k, "v": v, "k_exponent": ke, "v_exponent": ve}


def _handle(c, s):
  """What a user's program makes once and keeps."""
  sa = _library()
  if c["op"] == "rotary":
    return sa.make_rotary(c["head_dim"], _sections(c), pairing="adjacent" if c["adjacent"] else "half",
                          q_scale=c["head_dim"] ** -0.5)
  if c["op"] in ("write", "read"):
    return sa.KVCache(**s["cache"])
  if c["op"] == "attend":
    return (sa.make_splash_cached(window_left=None if c["window"] < 0 else c["window"], num_sinks=c["sinks"],
                                  attn_logits_soft_cap=c["cap"] or None, mask_value=-math.inf), sa.KVCache(**s["cache"]))
  mask = sa.LocalMask((c["n"], c["kv_len"] or c["n"]), (c["window"], 0), (c["kv_len"] or c["n"]) - c["n"], num_sinks=c["sinks"])
  return sa.make_splash_mha(mask, attn_logits_soft_cap=c["cap"] or None)


def prepare(case, seed):
  c, g = case, _generator(seed)
  s = {"case": c}
  if c["op"] == "rotary":
    s["q"], s["k"] = _heads_of(c, g, c["heads"]), _heads_of(c, g, c["kv_heads"])
    s["positions"] = _positions(c, seed)
    if c["train"]:
      s["d_out"] = tuple(torch.randn(x.shape, generator=g, device=DEVICE, dtype=x.dtype) for x in (s["q"], s["k"]))
      s["q"], s["k"] = (x.requires_grad_(True) for x in (s["q"], s["k"]))
  elif c["op"] == "sinks":
    kv = (c["batch"], c["kv_heads"], c["kv_len"] or c["n"], c["head_dim"])
    qs = (c["batch"], c["heads"], c["n"], c["head_dim"])
    normal = lambda shape: torch.randn(shape, generator=g, device=DEVICE)
    s["q"], s["k"], s["v"] = ((normal(qs) * c["head_dim"] ** -0.5).to(_dtype(c)), normal(kv).to(_dtype(c)), normal(kv).to(_dtype(c)))
    if c["train"]:
      s["d_out"] = normal(qs).to(_dtype(c))
      s["q"], s["k"], s["v"] = (x.requires_grad_(True) for x in (s["q"], s["k"], s["v"]))
  else:
    before, new = _lengths(c, seed)
    total = before + new
    if c["op"] == "read":
      total = before
    s["table"], pages = _table(c, c["max_len"] + (0 if c["op"] == "read" else c["n"]), g)
    s["cache"] = _cache(c, pages, g, filled=c["op"] != "write")
    device = lambda x: torch.from_numpy(x.astype(np.int32)).to(DEVICE)
    s["start"], s["counts"], s["lengths"] = device(before), device(new) if c["ragged_new"] else None, device(total)
    s["max_len"] = c["max_len"] if c["op"] == "read" else max(1, int(total.max()))
    if c["op"] == "write":
      s["k"], s["v"] = _heads_of(c, g, c["kv_heads"]), _heads_of(c, g, c["kv_heads"])
    elif c["op"] == "attend":
      qs = (c["batch"], c["heads"], c["n"], c["head_dim"])
      s["q"] = (torch.randn(qs, generator=g, device=DEVICE) * c["head_dim"] ** -0.5).to(_dtype(c))
      s["parents"] = torch.from_numpy(_parents(c, seed)).to(DEVICE) if c["tree"] else None
  if own:
    s["handle"] = _handle(c, s)
  return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------


def _quantize(x):
  """e4m3 codes and exponents e: x = code * 2^e per row of head_dim elements, e the smallest whole number with max|x| <= 448 * 2^e."""
  x = x.float()
  m, e = torch.frexp(x.abs().amax(-1))  # m in [0.5, 1), or 0
  e = (e - 9 + (m > 0.875)).clamp(MIN_EXPONENT, MAX_EXPONENT)  # 448 = 0.875 * 2^9
  e = torch.where(m > 0, e, MIN_EXPONENT)
  return torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn), e.to(torch.int8)


def _rows(s, index):
  """Rows [batch, kv_heads, tokens] of the flattened cache that hold the tokens `index` [batch, tokens] of each sequence."""
  c = s["case"]
  page = torch.gather(s["table"].long(), 1, index // c["page"])
  head = torch.arange(c["kv_heads"], device=DEVICE)[None, :, None]
  return (page[:, None] * c["kv_heads"] + head) * c["page"] + (index % c["page"])[:, None]


def _bytes(x):
  return x.view(-1, x.shape[-1]) if x.element_size() > 1 else x.view(torch.uint8).view(-1, x.shape[-1])


def _plain_write(s):
  c, cache = s["case"], s["cache"]
  token = torch.arange(c["n"], device=DEVICE)[None]
  index = s["start"].long()[:, None] + token
  live = (token < s["counts"][:, None]) if s["counts"] is not None else torch.ones_like(index, dtype=torch.bool)
  rows = _rows(s, torch.where(live, index, torch.zeros_like(index)))
  live = live[:, None].expand(rows.shape)
  for name in ("k", "v"):
    x = s[name]
    if c["quantized"]:
      x, e = _quantize(x)
      cache[name + "_exponent"].view(-1)[rows[live]] = e[live]
    _bytes(cache[name])[rows[live]] = x.view(torch.uint8)[live] if c["quantized"] else x[live]
  return _cache_out(s)


def _cache_out(s):
  return [x for x in (s["cache"][n] for n in ("k", "v", "k_exponent", "v_exponent")) if x is not None]


def _gathered(s, name, tokens):
  """[batch, kv_heads, tokens, head_dim] in 32 bits out of the cache."""
  index = torch.arange(tokens, device=DEVICE)[None].expand(s["case"]["batch"], tokens)
  rows = _rows(s, index)
  x = s["cache"][name].view(-1, s["case"]["head_dim"])
  if not s["case"]["quantized"]:
    return x[rows].float()
  x = x.view(torch.uint8)[rows].view(torch.float8_e4m3fn).float()
  return x * torch.exp2(s["cache"][name + "_exponent"].view(-1)[rows].float())[..., None]


def _plain_read(s):
  dead = torch.arange(s["max_len"], device=DEVICE)[None] >= s["lengths"][:, None]
  return tuple(_gathered(s, n, s["max_len"]).masked_fill(dead[:, None, :, None], 0.0).to(_dtype(s["case"])) for n in ("k", "v"))


def _ancestors(parents):
  """[batch, n, n] whether node j is node i or above it, by squaring the relation."""
  n = parents.shape[1]
  up = torch.eye(n, device=parents.device) + (parents[:, :, None] == torch.arange(n, device=parents.device)).float()
  for _ in range(max(1, math.ceil(math.log2(n)))):
    up = (up @ up > 0).float()
  return up > 0


def _seen(s, tokens):
  """[batch, 1, n, tokens] which cached tokens each new token sees."""
  c = s["case"]
  length = s["lengths"].long()[:, None, None]
  new = (s["counts"].long() if s["counts"] is not None else torch.full((c["batch"],), c["n"], device=DEVICE))[:, None, None]
  before = length - new
  key = torch.arange(tokens, device=DEVICE)[None, None]
  node = torch.arange(c["n"], device=DEVICE)[None, :, None]
  if c["tree"]:
    up = _ancestors(s["parents"])
    depth = up.sum(-1) - 1
    drafted = (key - before).clamp(0, c["n"] - 1).expand(c["batch"], c["n"], tokens)
    seen = (key < before) | ((key < length) & torch.gather(up, 2, drafted))
    position = before + depth[:, :, None]
    key = torch.where(key < before, key, before + torch.gather(depth[:, None].expand(-1, c["n"], -1), 2, drafted))
  else:
    position = before + node
    seen = key <= position
  if c["window"] >= 0:
    seen = seen & ((key >= position - c["window"]) | (key < c["sinks"]))
  return (seen & (node < new))[:, None]


def _softmax_products(c, q, k, v, seen):
  """Attention of q [batch, heads, rows, d] with the visibility `seen` [..., rows, keys] (rows that see nothing: zeros): out, the
  logarithm of the sums, and what a backward pass wants; the heads of a group share their kv head's products."""
  rows = q.shape[2]
  grouped = lambda x: x.reshape(x.shape[0], c["kv_heads"], -1, x.shape[-1])  # [batch, kv_heads, heads of a group * rows, ...]
  s = grouped(q) @ k.transpose(-1, -2)
  slope = None
  if c["cap"]:
    t = torch.tanh(s / c["cap"])
    s, slope = t * c["cap"], 1 - t * t
  s = s.unflatten(2, (-1, rows)).masked_fill(~seen.unsqueeze(-3), -math.inf).flatten(2, 3)
  m = s.amax(-1, keepdim=True)
  m = torch.where(m == -math.inf, torch.zeros_like(m), m)
  p = torch.exp(s - m)
  total = p.sum(-1, keepdim=True)
  p = p / torch.where(total > 0, total, torch.ones_like(total))
  return (p @ v).view(q.shape), (m + torch.log(total)).view(q.shape[:3]), p, slope, grouped


def _plain_attend(s):
  c = s["case"]
  k, v = (_gathered(s, n, s["max_len"]) for n in ("k", "v"))
  dead = (torch.arange(s["max_len"], device=DEVICE)[None] >= s["lengths"][:, None])[:, None, :, None]
  out, lse = _softmax_products(c, s["q"].float(), k, v.masked_fill(dead, 0.0), _seen(s, s["max_len"]))[:2]
  out = out.to(_dtype(c))
  return (out, lse) if c["lse"] else out


def _sinks_seen(c):
  kv = c["kv_len"] or c["n"]
  position = torch.arange(c["n"], device=DEVICE)[:, None] + (kv - c["n"])
  key = torch.arange(kv, device=DEVICE)[None]
  return (key <= position) & ((key >= position - c["window"]) | (key < c["sinks"]))


def _plain_sinks(s):
  c = s["case"]
  with torch.no_grad():
    q = s["q"].float()
    k, v = s["k"].float(), s["v"].float()
    out, _, p, slope, grouped = _softmax_products(c, q, k, v, _sinks_seen(c))
    if not c["train"]:
      return out.to(_dtype(c))
    do = grouped(s["d_out"].float())
    dv = p.transpose(-1, -2) @ do
    ds = (do @ v.transpose(-1, -2)).sub_((do * grouped(out)).sum(-1, keepdim=True)).mul_(p)
    if slope is not None:
      ds = ds.mul_(slope)
    return tuple(x.to(_dtype(c)) for x in (out, (ds @ k).view(q.shape), ds.transpose(-1, -2) @ grouped(q), dv))


def _angles(c, positions):
  """[batch, 1, n, pairs] in 64 bits: position on the pair's axis times 10000^(-2 i / head_dim)."""
  pairs = c["head_dim"] // 2
  axis = torch.repeat_interleave(torch.arange(c["axes"]), torch.tensor(_sections(c))).to(DEVICE)
  p = positions.unsqueeze(1) if c["axes"] == 1 else positions
  frequency = 10000.0 ** (torch.arange(pairs, device=DEVICE, dtype=torch.float64) * (-2.0 / c["head_dim"]))
  return (p.double()[:, axis].transpose(1, 2) * frequency)[:, None]


def _split(c, x):
  return (x[..., 0::2], x[..., 1::2]) if c["adjacent"] else x.chunk(2, -1)


def _joined(c, a, b):
  return torch.stack((a, b), -1).flatten(-2) if c["adjacent"] else torch.cat((a, b), -1)


def _turn(c, x, cos, sin, scale):
  a, b = _split(c, x)
  return _joined(c, a * cos - b * sin, b * cos + a * sin) * scale


def _plain_rotary(s):
  c = s["case"]
  with torch.no_grad():
    angle = _angles(c, s["positions"])
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    scale = c["head_dim"] ** -0.5
    dtype = _dtype(c)
    out = [_turn(c, s["q"].float(), cos, sin, scale).to(dtype), _turn(c, s["k"].float(), cos, sin, 1.0).to(dtype)]
    if c["train"]:
      out += [_turn(c, s["d_out"][0].float(), cos, -sin, scale).to(dtype), _turn(c, s["d_out"][1].float(), cos, -sin, 1.0).to(dtype)]
    return tuple(out)


# ---------------------------------------------------------------------------


def _own(s):
  c, handle = s["case"], s["handle"]
  if c["op"] == "rotary":
    q, k = handle(s["q"], s["k"], s["positions"])
    if not c["train"]:
      return q, k
    return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (s["q"], s["k"]), s["d_out"])
  if c["op"] == "write":
    handle.write(s["k"], s["v"], s["table"], s["start"], counts=s["counts"])
    return _cache_out(s)
  if c["op"] == "read":
    return handle.read(s["table"], s["lengths"], s["max_len"], dtype=_dtype(c))
  if c["op"] == "attend":
    attend, cache = handle
    out = attend(s["q"], cache, s["table"], s["lengths"], counts=s["counts"], parents=s["parents"], save_residuals=c["lse"])
    return (out[0], out[1][0]) if c["lse"] else out
  out = handle(s["q"], s["k"], s["v"])
  if not c["train"]:
    return out
  return (out.detach(),) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["d_out"])


def run(state):
  if own:
    return _own(state)
  return {"rotary": _plain_rotary, "write": _plain_write, "read": _plain_read, "attend": _plain_attend,
          "sinks": _plain_sinks}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------


def work(case):
  """With the lengths of seed 0: other seeds draw others of the same range."""
  c = case
  d = c["head_dim"]
  row = d + 1 if c["quantized"] else 2 * d
  if c["op"] == "rotary":
    numbers = c["batch"] * c["n"] * (c["heads"] + c["kv_heads"]) * d
    passes = 2 if c["train"] else 1
    return {"bytes": passes * (4 * numbers + 4 * c["batch"] * c["axes"] * c["n"]), "flops": passes * 3 * numbers}
  before, new = _lengths(c, 0)
  if c["op"] in ("write", "read"):
    rows = 2 * c["kv_heads"] * int((new if c["op"] == "write" else before).sum())
    zeros = 2 * c["kv_heads"] * (c["batch"] * c["max_len"] - int(before.sum())) if c["op"] == "read" else 0
    return {"bytes": rows * (row + 2 * d) + zeros * 2 * d, "flops": 2 * rows * d}
  if c["op"] == "attend":
    pairs, keys = 0, 0
    for b, m in zip(before.tolist(), new.tolist()):
      seen = min(b, c["window"] + min(c["sinks"], max(0, b - c["window"]))) if c["window"] >= 0 else b
      keys += seen + m if m else 0
      pairs += m * (seen + (m + 1) / 2)
    q = c["batch"] * c["heads"] * c["n"] * d
    return {"bytes": 2 * c["kv_heads"] * keys * row + 4 * q + (q // d * 4 if c["lse"] else 0), "flops": 4 * d * c["heads"] * pairs}
  kv = c["kv_len"] or c["n"]
  i = np.arange(c["n"]) + kv - c["n"]
  lo = np.maximum(0, i - c["window"])
  pairs = c["batch"] * c["heads"] * int((i + 1 - lo + np.minimum(lo, c["sinks"])).sum())
  q, k = c["batch"] * c["heads"] * c["n"] * d * 2, c["batch"] * c["kv_heads"] * kv * d * 2
  return {"bytes": (4 if c["train"] else 2) * (q + k), "flops": (14 if c["train"] else 4) * d * pairs}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, written apart from the forms above
# ---------------------------------------------------------------------------


def _exact_rows(s, name, b, tokens):
  """Tokens 0..tokens-1 of sequence b in 64 bits, [kv_heads, tokens, head_dim]."""
  c = s["case"]
  pages = s["table"][b, :-(-tokens // c["page"])].long()
  x = s["cache"][name][pages].double()
  if c["quantized"]:
    x = x * 2.0 ** s["cache"][name + "_exponent"][pages].double().unsqueeze(-1)
  return x.transpose(0, 1).reshape(c["kv_heads"], -1, c["head_dim"])[:, :tokens]


def _exact_attend(s):
  c = s["case"]
  out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
  lse = torch.full(out.shape[:3], -math.inf, dtype=torch.float64, device=DEVICE)
  lengths = s["lengths"].tolist()
  counts = s["counts"].tolist() if s["counts"] is not None else [c["n"]] * c["batch"]
  parents = s["parents"].tolist() if c["tree"] else None
  group = c["heads"] // c["kv_heads"]
  for b in range(c["batch"]):
    length, m = lengths[b], counts[b]
    if m == 0:
      continue
    before = length - m
    seen = np.zeros((m, length), bool)
    depth = np.zeros(m, np.int64)
    for i in range(m):
      above = [i] if c["tree"] else list(range(i, -1, -1))
      while c["tree"] and parents[b][above[-1]] >= 0:
        above.append(parents[b][above[-1]])
      depth[i] = len(above) - 1
      position = before + depth[i]
      first = max(0, position - c["window"]) if c["window"] >= 0 else 0
      seen[i, first:before] = True
      seen[i, :min(c["sinks"], before)] = True
      for j in above:
        if before + depth[j] >= first or before + depth[j] < c["sinks"]:
          seen[i, before + j] = True
    seen = torch.from_numpy(seen).to(DEVICE)
    k, v = (_exact_rows(s, n, b, length) for n in ("k", "v"))
    q = s["q"][b].double()[:, :m].reshape(c["kv_heads"], group * m, -1)
    x = torch.bmm(q, k.transpose(1, 2))
    if c["cap"]:
      x = c["cap"] * torch.tanh(x / c["cap"])
    x = torch.where(seen.repeat(group, 1)[None], x, torch.tensor(-math.inf, dtype=torch.float64, device=DEVICE))
    z = torch.logsumexp(x, -1)
    out[b, :, :m] = torch.bmm(torch.exp(x - z[..., None]), v).reshape(c["heads"], m, -1)
    lse[b, :, :m] = z.reshape(c["heads"], m)
  return (out, lse) if c["lse"] else out


def _exact_sinks(s):
  c = s["case"]
  kv, group = c["kv_len"] or c["n"], c["heads"] // c["kv_heads"]
  q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
  out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
  do = s["d_out"].double() if c["train"] else None
  i = torch.arange(kv - c["n"], kv, device=DEVICE).unsqueeze(1)
  j = torch.arange(kv, device=DEVICE)
  hidden = (j > i) | ((i - j > c["window"]) & (j >= c["sinks"]))
  for b in range(c["batch"]):
    for h in range(c["heads"]):
      kh, vh = k[b, h // group], v[b, h // group]
      x = q[b, h] @ kh.T
      if c["cap"]:
        t = torch.tanh(x / c["cap"])
        x = c["cap"] * t
      p = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
      out[b, h] = p @ vh
      if c["train"]:
        dv[b, h // group] += p.T @ do[b, h]
        g = p * (do[b, h] @ vh.T - (out[b, h] * do[b, h]).sum(1, keepdim=True))
        if c["cap"]:
          g = g * (1 - t.square())
        dq[b, h] = g @ kh
        dk[b, h // group] += g.T @ q[b, h]
  return (out, dq, dk, dv) if c["train"] else out


def _exact_rotary(s):
  c = s["case"]
  sections, pairs = _sections(c), c["head_dim"] // 2
  positions = s["positions"].double().reshape(c["batch"], c["axes"], c["n"])
  angle = torch.empty(c["batch"], 1, c["n"], pairs, dtype=torch.float64, device=DEVICE)
  i = 0
  for axis, count in enumerate(sections):
    for _ in range(count):
      angle[:, 0, :, i] = positions[:, axis] * math.exp(-2 * i / c["head_dim"] * math.log(10000.0))
      i += 1
  turn = torch.polar(torch.ones_like(angle), angle)

  def rotated(x, turn, scale):
    x = x.detach().double()
    x = x.unflatten(-1, (pairs, 2)) if c["adjacent"] else x.unflatten(-1, (2, pairs)).transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(x.contiguous()) * turn) * scale
    return (y if c["adjacent"] else y.transpose(-1, -2)).flatten(-2)

  scale = 1 / math.sqrt(c["head_dim"])
  out = (rotated(s["q"], turn, scale), rotated(s["k"], turn, 1.0))
  if c["train"]:
    out += (rotated(s["d_out"][0], turn.conj(), scale), rotated(s["d_out"][1], turn.conj(), 1.0))
  return out


def exact(case, seed):
  c = case
  if c["op"] == "write":
    return None  # codes and copies: equal, or not
  s = prepare(c, seed)
  if c["op"] == "attend":
    return _exact_attend(s)
  if c["op"] == "sinks":
    return _exact_sinks(s)
  if c["op"] == "rotary":
    return _exact_rotary(s)
  out = []
  for name in ("k", "v"):
    x = torch.zeros(c["batch"], c["kv_heads"], s["max_len"], c["head_dim"], dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(s["lengths"].tolist()):
      x[b, :, :n] = _exact_rows(s, name, b, n)
    out.append(x)
  return tuple(out)
