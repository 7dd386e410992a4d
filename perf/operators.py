"""The operators of a KV cache held in 8 or 4 bits, as cases that can be timed and checked: rotating and quantising keys and
values as they are written and reading pages back ("store"), attention of single tokens ("decode") and of prompts ("prompt").

The format: a head's row in groups of 32 dims, each with one power of two as its scale (a byte, the exponent + 127; 255: the
group reads back as NaN) and elements of e2m1 ("mxfp4") or e4m3 ("mxfp8").  The exponent is the smallest with
absmax <= 7 (464) * 2^e, from -100 to 125 (119); elements are rounded to the nearest, ties to even, and clamped.

A page of one KV head is one run of bytes, 64 keys of elements and then their scales:
  keys:    elements row by row (4 bits: even dim low); scale of key 32 a + 8 b + 4 c + d, group j at 64 j + 4 (4 b + d) + 2 a + c
  values:  units of 16 bytes, those of dims 2 r and 2 r + 1 of every group side by side: [64 / n][16 r][n keys][Dh / 32 groups]
           of a byte (4 bits: even dim low) or two, n as fits; scales [64 keys][Dh / 32]
"""
import math
import random

import torch

own = False  # the kernels' side, imported where it is asked for

DEV = "cuda:0"
PAGE = 64
LOW = -100
EMAX = {"mxfp4": 2, "mxfp8": 8}  # exponent of the largest element
TOP = {"mxfp4": 7.0, "mxfp8": 464.0}
MOST = {"mxfp4": 6.0, "mxfp8": 448.0}
HIGH = {"mxfp4": 125, "mxfp8": 119}


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
  def store(name, fmt, H, Hkv, Dh, B, lo, hi, past):
    return {"name": name, "path": "store", "fmt": fmt, "H": H, "Hkv": Hkv, "Dh": Dh, "batch": B, "lo": lo, "hi": hi, "past": past}

  def decode(name, fmt, H, Hkv, Dh, B, lo, hi):
    return {"name": name, "path": "decode", "fmt": fmt, "H": H, "Hkv": Hkv, "Dh": Dh, "batch": B, "lo": lo, "hi": hi}

  def prompt(name, fmt, H, Hkv, Dh, B, lo, hi, past):
    return {"name": name, "path": "prompt", "fmt": fmt, "H": H, "Hkv": Hkv, "Dh": Dh, "batch": B, "lo": lo, "hi": hi, "past": past}
  return [
    # one decode step of 64 requests: a token each, far into their contexts, and the pages they went to
    store("store_step_64", "mxfp4", 64, 8, 128, 64, 1, 1, 2000),
    # prompts of unlike length that arrive together, some of them continuing a cached prefix
    store("store_prompts_9", "mxfp8", 32, 8, 128, 9, 60, 500, 90),
    # one long document
    store("store_doc_8191", "mxfp4", 32, 8, 128, 1, 8191, 8191, 0),
    # a chat of one user: latency counts
    decode("decode_1x700", "mxfp4", 32, 8, 128, 1, 700, 700),
    # a server's ordinary step, contexts of all lengths
    decode("decode_64_ragged", "mxfp8", 32, 8, 128, 64, 30, 2000),
    # a full batch of the 70B model's heads
    decode("decode_512x525", "mxfp4", 64, 8, 128, 512, 520, 530),
    # long documents, few of them: the work has to be split along the contexts
    decode("decode_8x32k", "mxfp4", 32, 8, 128, 8, 31000, 32700),
    # heads of 64
    decode("decode_256_d64", "mxfp4", 32, 8, 64, 256, 100, 1500),
    # every head with keys and values of its own
    decode("decode_48_mha", "mxfp8", 32, 32, 128, 48, 200, 700),
    # the next turns of a few chats: short questions behind cached contexts
    prompt("prompt_4_turns", "mxfp4", 32, 8, 128, 4, 5, 60, 1500),
    # prompts of unlike length
    prompt("prompt_8_ragged", "mxfp8", 64, 8, 128, 8, 100, 900, 0),
    # one long prompt
    prompt("prompt_1x4096", "mxfp4", 32, 8, 128, 1, 4096, 4096, 0),
  ]


def _log(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  path = rng.choice(["store", "decode", "decode", "prompt"])
  H, Hkv, Dh = rng.choice([(64, 8, 128), (32, 8, 128), (32, 8, 64), (32, 32, 128), (14, 2, 64), (28, 4, 128)])
  c = {"path": path, "fmt": rng.choice(["mxfp4", "mxfp8"]), "H": H, "Hkv": Hkv, "Dh": Dh}
  if path == "store":
    B = _log(rng, 1, 256)
    hi = _log(rng, 1, max(1, 8000 // B))
    return c | {"batch": B, "lo": max(1, hi // rng.choice([1, 2, 5])), "hi": hi, "past": rng.choice([0, _log(rng, 1, 3000)])}
  if path == "decode":
    B = _log(rng, 1, 512)
    hi = _log(rng, 20, min(32000, max(40, 260000 * 8 // (Hkv * B))))
    return c | {"batch": B, "lo": max(1, hi // rng.choice([1, 1, 2, 10])), "hi": hi}
  B = _log(rng, 1, 12)
  hi = _log(rng, 2, min(3000, 6000 // B))
  return c | {"batch": B, "lo": max(1, hi // rng.choice([1, 2, 5])), "hi": hi, "past": rng.choice([0, _log(rng, 1, 1500 if B < 6 else 300)])}


def _sizes(case, seed):
  """Tokens that come new and contexts including them, per sequence: the case's lengths, single tokens' in the seed's order."""
  B, path = case["batch"], case["path"]
  r = random.Random("%d %d %d" % (B, case["lo"], case["hi"]))
  n = [r.randint(case["lo"], case["hi"]) for _ in range(B)]
  if path == "decode":
    random.Random(seed).shuffle(n)
    return [1] * B, n
  past = [r.randint(case["past"] // 2, case["past"]) if case["past"] else 0 for _ in range(B)]
  return n, [a + b for a, b in zip(n, past)]


def work(case):
  H, Hkv, Dh = case["H"], case["Hkv"], case["Dh"]
  new, ctx = _sizes(case, 0)
  T = sum(new)
  row = 2 * Hkv * (Dh * (1 if case["fmt"] == "mxfp8" else 0.5) + Dh / 32)  # a token's keys and values in the cache
  if case["path"] == "store":  # projections read, queries and cache written; the pages touched read back and written in bf16
    back = sum((c - 1) % PAGE + 1 if n == 1 else c for n, c in zip(new, ctx))
    return {"bytes": T * 2 * ((H + 2 * Hkv) * Dh + H * Dh) + T * row + back * (row + 4 * Hkv * Dh), "flops": T * (H + 2 * Hkv) * Dh * 4}
  pairs = sum(n * c - n * (n - 1) // 2 for n, c in zip(new, ctx))
  return {"bytes": sum(ctx) * row + 4 * T * H * Dh, "flops": 4 * H * Dh * pairs}


# ---------------------------------------------------------------------------------------------------------- the format
def _order(device):
  """Where the scale of key i stands among its group's 64."""
  i = torch.arange(PAGE, device=device)
  return 4 * (4 * (i // 8 % 4) + i % 4) + 2 * (i // 32) + i // 4 % 2


def _encode(x, fmt):
  """x [..., Dh] fp32 -> element codes [..., Dh] uint8, scale bytes [..., Dh / 32] uint8."""
  g = x.unflatten(-1, (-1, 32))
  a = g.abs().amax(-1)
  bad = ~torch.isfinite(a)
  m, e = torch.frexp(torch.where(bad, torch.ones_like(a), a))
  e = e - 1 - EMAX[fmt]
  e = e + (m * 2.0 ** (EMAX[fmt] + 1) > TOP[fmt]).to(e.dtype)
  e = torch.where(a > 0, e, torch.full_like(e, LOW)).clamp(LOW, HIGH[fmt])
  y = (g * ((127 - e) << 23).view(torch.float32)[..., None]).clamp(-MOST[fmt], MOST[fmt])
  if fmt == "mxfp8":
    code = y.to(torch.float8_e4m3fn).view(torch.uint8)
  else:
    w = y.abs()
    step = torch.exp2((torch.frexp(w)[1] - 1).clamp(min=0).float()) * 0.5
    w = torch.round(w / step) * step
    w = w.clamp(max=6.0)
    code = torch.where(w <= 2, w * 2, torch.where(w <= 4, w + 2, w + 1)).to(torch.uint8) + 8 * (y < 0).to(torch.uint8)
  code = torch.where(bad[..., None], torch.zeros_like(code), code)
  return code.flatten(-2), torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def _value(code, scale, fmt):
  """Element codes [..., Dh], scale bytes [..., Dh / 32] -> fp32 values [..., Dh]."""
  s = (scale.int() << 23).view(torch.float32)
  s = torch.where(scale == 255, torch.full_like(s, float("nan")), s)
  if fmt == "mxfp8":
    v = code.view(torch.float8_e4m3fn).float()
  else:
    n = (code & 7).float()
    v = torch.where(n <= 4, n * 0.5, torch.where(n <= 6, n - 2, n - 1)) * torch.where(code >= 8, -1.0, 1.0)
  return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _pack_pages(kcode, kscale, vcode, vscale, fmt):
  """Codes [n, Hkv, 64, Dh] and scales [n, Hkv, 64, J] of whole pages -> the caches' bytes [n, Hkv, page bytes]."""
  n, G, _, Dh = kcode.shape
  J = Dh // 32
  ke = kcode if fmt == "mxfp8" else kcode[..., 0::2] | (kcode[..., 1::2] << 4)
  ks = torch.empty(n, G, J, PAGE, dtype=torch.uint8, device=kcode.device)
  ks[..., _order(kcode.device)] = kscale.transpose(2, 3)
  v = vcode.view(n, G, PAGE, J, 16, 2)  # [key, group, r, even / odd]
  v = v if fmt == "mxfp8" else v[..., :1] | (v[..., 1:] << 4)
  per = 16 // (J * v.shape[-1])
  v = v.unflatten(2, (PAGE // per, per)).permute(0, 1, 2, 5, 3, 4, 6)  # [unit, r, key, group, bytes]
  return (torch.cat([ke.flatten(2), ks.flatten(2)], -1), torch.cat([v.flatten(2), vscale.flatten(2)], -1))


def _unpack_pages(k, v, Dh, fmt):
  """The inverse: pages' bytes -> keys and values [n, Hkv, 64, Dh] fp32."""
  n, G = k.shape[:2]
  J, e = Dh // 32, PAGE * Dh // (1 if fmt == "mxfp8" else 2)
  ke = k[..., :e].view(n, G, PAGE, -1)
  kcode = ke if fmt == "mxfp8" else torch.stack([ke & 15, ke >> 4], -1).flatten(-2)
  kscale = k[..., e:].view(n, G, J, PAGE)[..., _order(k.device)].transpose(2, 3)
  w = 2 if fmt == "mxfp8" else 1
  per = 16 // (J * w)
  ve = v[..., :e].view(n, G, PAGE // per, 16, per, J, w).permute(0, 1, 2, 4, 5, 3, 6).reshape(n, G, PAGE, J, 16, w)
  vcode = ve if fmt == "mxfp8" else torch.cat([ve & 15, ve >> 4], -1)
  return _value(kcode.contiguous(), kscale, fmt), _value(vcode.reshape(n, G, PAGE, Dh).contiguous(), v[..., e:].view(n, G, PAGE, J), fmt)


# ---------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
  H, Hkv, Dh, fmt, B = case["H"], case["Hkv"], case["Dh"], case["fmt"], case["batch"]
  new, ctx = _sizes(case, seed)
  g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)
  pages = [-(-c // PAGE) for c in ctx]
  width, total = max(pages), sum(pages)
  pool = total + 3
  chan = torch.exp(0.5 * torch.randn(Hkv, 1, Dh, generator=g, device=DEV))  # keys have loud and quiet channels
  order = torch.randperm(pool, generator=g, device=DEV)[:total].to(torch.int32)
  tables = torch.zeros(B, width, dtype=torch.int32, device=DEV)
  valid = torch.arange(width, device=DEV)[None] < torch.tensor(pages, device=DEV)[:, None]
  tables[valid] = order
  k = torch.randn(pool, Hkv, PAGE, Dh, generator=g, device=DEV) * chan
  v = torch.randn(pool, Hkv, PAGE, Dh, generator=g, device=DEV)
  kc, vc = _pack_pages(*_encode(k, fmt), *_encode(v, fmt), fmt)
  del k, v
  s = {"path": case["path"], "fmt": fmt, "H": H, "Hkv": Hkv, "Dh": Dh, "k": kc.contiguous(), "v": vc.contiguous(), "tables": tables,
       "ctx": torch.tensor(ctx, dtype=torch.int32, device=DEV), "scale": 1.0 / math.sqrt(Dh)}
  T = sum(new)
  if case["path"] == "store":
    pos = torch.cat([torch.arange(c - n, c, device=DEV) for n, c in zip(new, ctx)])
    seq = torch.repeat_interleave(torch.arange(B, device=DEV), torch.tensor(new, device=DEV))
    s["slots"] = tables[seq, pos // PAGE].long() * PAGE + pos % PAGE
    s["pos"] = pos.int()
    x = torch.randn(T, H + 2 * Hkv, Dh, generator=g, device=DEV)
    x[:, H:H + Hkv] *= chan[:, 0]
    s["qkv"] = x.to(torch.bfloat16).flatten(1)
    rows = max(ctx)
    ang = torch.arange(rows, dtype=torch.float64)[:, None] / 500000.0 ** (torch.arange(0, Dh, 2, dtype=torch.float64) / Dh)
    s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], 1).float().to(DEV)
    if case["hi"] == 1:  # single tokens: the one page each went to
      s["tables"] = tables.gather(1, ((s["ctx"] - 1) // PAGE).long()[:, None]).contiguous()
      s["ctx"] = (s["ctx"] - 1) % PAGE + 1
    return s
  s["q"] = (2.0 * torch.randn(T, H, Dh, generator=g, device=DEV)).to(torch.bfloat16)
  if case["path"] == "prompt":
    cu = [0]
    for n in new:
      cu.append(cu[-1] + n)
    s["cu"], s["max_new"] = torch.tensor(cu, dtype=torch.int32, device=DEV), max(new)
  elif own:
    from xotorch_support_jetson_amd.ops import kernels as K
    s["ws"] = K.MXDecodeWorkspace(B, H, Hkv, Dh, width * PAGE, DEV)
  return s


# ---------------------------------------------------------------------------------------------------------- one pass
def run(s):
  if own:
    from xotorch_support_jetson_amd.ops import kernels as K
    if s["path"] == "store":
      q = K.rope_kv_write_mx(s["qkv"], s["pos"], s["cos_sin"], s["slots"], s["k"], s["v"], s["H"], s["Hkv"])
      return (q,) + K.kv_read_mx(s["k"], s["v"], s["tables"], s["ctx"], s["Dh"])
    if s["path"] == "decode":
      return K.attn_decode_mx(s["q"], s["k"], s["v"], s["tables"], s["ctx"], s["scale"], s["ws"])
    return K.attn_prefill_mx(s["q"], s["k"], s["v"], s["tables"], s["cu"], s["ctx"], s["max_new"], s["scale"])
  return {"store": _store, "decode": _decode, "prompt": _prompt}[s["path"]](s)


def _rows(s):
  """The step's pages as fp32 keys and values [B, Hkv, width * 64, Dh], zeros past the contexts."""
  B, W = s["tables"].shape
  t = s["tables"].long().flatten()
  k, v = _unpack_pages(s["k"][t], s["v"][t], s["Dh"], s["fmt"])
  live = (torch.arange(W * PAGE, device=DEV)[None] < s["ctx"][:, None])[:, None, :, None]
  k, v = (x.view(B, W, s["Hkv"], PAGE, s["Dh"]).transpose(1, 2).reshape(B, s["Hkv"], W * PAGE, s["Dh"]) for x in (k, v))
  return torch.where(live, k, torch.zeros((), device=DEV)), torch.where(live, v, torch.zeros((), device=DEV))


def _store(s):
  H, Hkv, Dh, fmt = s["H"], s["Hkv"], s["Dh"], s["fmt"]
  x = s["qkv"].view(-1, H + 2 * Hkv, Dh).float()
  cs = s["cos_sin"][s["pos"].long()][:, None]
  c, sn = cs[..., :Dh // 2], cs[..., Dh // 2:]
  lo, hi = x[:, :H + Hkv, :Dh // 2], x[:, :H + Hkv, Dh // 2:]
  rot = torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1)
  # the new rows go among the bytes of the pages they belong to
  page, off = s["slots"] // PAGE, s["slots"] % PAGE
  J, w = Dh // 32, 2 if fmt == "mxfp8" else 1
  e, per = PAGE * Dh * w // 2, 16 // (J * w)
  kcode, kscale = _encode(rot[:, H:], fmt)
  vcode, vscale = _encode(x[:, H + Hkv:], fmt)
  pool = s["k"].shape[0]
  s["k"][..., :e].view(pool, Hkv, PAGE, -1)[page, :, off] = kcode if fmt == "mxfp8" else kcode[..., 0::2] | (kcode[..., 1::2] << 4)
  s["k"][..., e:].view(pool, Hkv, J, PAGE)[page, :, :, _order(DEV)[off]] = kscale
  vb = vcode.unflatten(-1, (J, 16, 2)).transpose(2, 3)  # [T, head, r, group, even / odd]
  vb = vb if fmt == "mxfp8" else vb[..., :1] | (vb[..., 1:] << 4)
  s["v"][..., :e].view(pool, Hkv, PAGE // per, 16, per, J * w)[page, :, off // per, :, off % per] = vb.flatten(3)
  s["v"][..., e:].view(pool, Hkv, PAGE, J)[page, :, off] = vscale
  k, v = _rows(s)
  B, W = s["tables"].shape
  k, v = (t.to(torch.bfloat16).view(B, Hkv, W, PAGE, Dh).transpose(1, 2).reshape(B * W, Hkv, PAGE, Dh) for t in (k, v))
  v = v.unflatten(2, (8, 8)).transpose(3, 4).reshape(B * W, Hkv, Dh, PAGE)  # (8 keys of a dim side by side)
  return rot[:, :H].to(torch.bfloat16), k, v


def _decode(s):
  k, v = _rows(s)
  B, H, Dh = s["q"].shape
  Hkv = s["Hkv"]
  q = s["q"].float().view(B, Hkv, H // Hkv, Dh)
  p = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
  dead = (torch.arange(k.shape[2], device=DEV)[None] >= s["ctx"][:, None])[:, None, None]
  p = p.masked_fill(dead, float("-inf"))
  p = torch.exp(p - p.amax(-1, keepdim=True))
  return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).view(B, H, Dh).to(torch.bfloat16)


def _prompt(s):
  k, v = _rows(s)
  T, H, Dh = s["q"].shape
  Hkv, B, m = s["Hkv"], s["ctx"].numel(), s["max_new"]
  row = torch.arange(T, device=DEV)
  b = torch.searchsorted(s["cu"][1:].contiguous(), row.int(), right=True)
  i = row - s["cu"].long()[b]
  q = torch.zeros(B, m, H, Dh, device=DEV)
  q[b, i] = s["q"].float()
  q = q.view(B, m, Hkv, H // Hkv, Dh).permute(0, 2, 3, 1, 4).reshape(B, Hkv, (H // Hkv) * m, Dh)
  p = (torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]).view(B, Hkv, H // Hkv, m, -1)
  n = s["cu"][1:] - s["cu"][:-1]
  last = (s["ctx"] - n)[:, None] + torch.arange(m, device=DEV)[None]  # the last key that a new token sees
  dead = torch.arange(k.shape[2], device=DEV)[None, None] > last[:, :, None]
  p = p.masked_fill(dead[:, None, None], float("-inf"))
  p = torch.exp(p - p.amax(-1, keepdim=True))
  o = torch.matmul(p.view(B, Hkv, (H // Hkv) * m, -1), v).view(B, Hkv, H // Hkv, m, Dh) / p.sum(-1, keepdim=True)
  return o.permute(0, 3, 1, 2, 4).reshape(B, m, H, Dh)[b, i].to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------------------- 64 bits
_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _e4m3(c):
  e, m = c >> 3 & 15, c & 7
  x = float("nan") if c & 127 == 127 else (1 + m / 8) * 2.0 ** (e - 7) if e else m / 8 * 2.0 ** -6
  return -x if c & 128 else x


def _levels(fmt):
  pos = _E2M1 if fmt == "mxfp4" else [_e4m3(c) for c in range(127)]
  return torch.tensor(pos, dtype=torch.float64, device=DEV)


def _nearest(x, fmt):
  """float64 rows [..., Dh] as the format holds them, by searching its levels."""
  lv = _levels(fmt)
  g = x.reshape(*x.shape[:-1], -1, 32)
  a = g.abs().amax(-1, keepdim=True)
  e = torch.ceil(torch.log2(a.clamp(min=2.0 ** -140) / TOP[fmt]))
  e = torch.where(a > TOP[fmt] * torch.exp2(e), e + 1, e)
  e = torch.where(a <= TOP[fmt] * torch.exp2(e - 1), e - 1, e).clamp(LOW, HIGH[fmt])
  y = (g.abs() / torch.exp2(e)).clamp(max=float(lv[-1]))
  up = torch.searchsorted(lv, y.contiguous()).clamp(max=lv.numel() - 1)
  dn = (up - 1).clamp(min=0)
  a, b = y - lv[dn], lv[up] - y
  pick = torch.where((a < b) | ((a == b) & (dn % 2 == 0)), dn, up)  # (a tie goes to the even code)
  return (lv[pick] * torch.exp2(e) * torch.sign(g)).reshape(x.shape)


def _cached(s, b):
  """Sequence b's keys and values [ctx, Hkv, Dh] in float64, byte by byte from tables of values."""
  Dh, fmt, n = s["Dh"], s["fmt"], int(s["ctx"][b])
  J = Dh // 32
  key = torch.arange(n, device=DEV)[:, None]
  page, off = s["tables"][b].long()[key // PAGE], key % PAGE
  d = torch.arange(Dh, device=DEV)[None]
  j, r, odd = d // 32, d % 32 // 2, d % 2
  e = PAGE * Dh // (2 if fmt == "mxfp4" else 1)
  codes = torch.tensor([(-x if c & 8 else x) for c, x in enumerate(_E2M1 * 2)] if fmt == "mxfp4" else [_e4m3(c) for c in range(256)],
                       dtype=torch.float64, device=DEV)
  if fmt == "mxfp4":
    per = 16 // J
    kat, vat, bits = off * (Dh // 2) + d // 2, ((off // per) * 16 + r) * 16 + off % per * J + j, 4 * odd
    pick = lambda x: (x.int() >> bits[..., None]) & 15  # noqa: E731
  else:
    per = 8 // J
    kat, vat = off * Dh + d, ((off // per) * 16 + r) * 16 + (off % per * J + j) * 2 + odd
    pick = lambda x: x.int()  # noqa: E731
  ksc = e + 64 * j + 4 * (4 * (off // 8 % 4) + off % 4) + 2 * (off // 32) + off // 4 % 2
  at = lambda t, i: t.transpose(1, 2)[page.expand_as(i), i]  # noqa: E731  [n, Dh, Hkv]
  value = lambda t, i, sc: (codes[pick(at(t, i)).long()] * torch.exp2(at(t, sc).double() - 127)).transpose(1, 2)  # noqa: E731
  return value(s["k"], kat, ksc), value(s["v"], vat, e + off * J + j)


def exact(case, seed):
  s = prepare(case, seed)
  H, Hkv, Dh = s["H"], s["Hkv"], s["Dh"]
  if s["path"] == "store":
    x = s["qkv"].double().view(-1, H + 2 * Hkv, Dh)
    c, sn = (t[:, None] for t in s["cos_sin"].double()[s["pos"].long()].split(Dh // 2, 1))
    a, b = x[:, :H + Hkv].split(Dh // 2, 2)
    rot = torch.cat([a * c - b * sn, a * sn + b * c], 2)
    kn, vn = _nearest(rot[:, H:], case["fmt"]), _nearest(x[:, H + Hkv:], case["fmt"])
    B, W = s["tables"].shape
    k = torch.zeros(B * W, Hkv, PAGE, Dh, dtype=torch.float64, device=DEV)
    v = torch.zeros_like(k)
    where = {}
    for i in range(B):
      for w, p in enumerate(s["tables"][i, :-(-int(s["ctx"][i]) // PAGE)].tolist()):
        where[p] = i * W + w
      n = int(s["ctx"][i])
      kb, vb = _cached(s, i)
      t = torch.arange(n, device=DEV)
      k[i * W + t // PAGE, :, t % PAGE], v[i * W + t // PAGE, :, t % PAGE] = kb, vb
    out = torch.full((s["k"].shape[0],), -1, dtype=torch.int64)
    for p, i in where.items():
      out[p] = i
    row = out.to(DEV)[s["slots"] // PAGE]
    k[row, :, s["slots"] % PAGE], v[row, :, s["slots"] % PAGE] = kn, vn
    return rot[:, :H], k, v.reshape(B * W, Hkv, 8, 8, Dh).transpose(3, 4).reshape(B * W, Hkv, Dh, PAGE)
  got = []
  cu = s["cu"].tolist() if s["path"] == "prompt" else list(range(case["batch"] + 1))
  for i in range(case["batch"]):
    k, v = _cached(s, i)
    q = s["q"][cu[i]:cu[i + 1]].double()
    n, m = k.shape[0], q.shape[0]
    o = torch.empty_like(q)
    see = torch.arange(n, device=DEV)[None] <= torch.arange(n - m, n, device=DEV)[:, None]
    for h in range(H):
      z = (q[:, h] @ k[:, h * Hkv // H].t()) * s["scale"]
      o[:, h] = torch.softmax(z.masked_fill(~see, float("-inf")), -1) @ v[:, h * Hkv // H]
    got.append(o)
  return torch.cat(got)
