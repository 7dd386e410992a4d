"""The KV cache in 8 or 4 bits (ops.kernels *_mx, csrc/kv_mx.hip): its format against a search of the levels, writing and reading back
against that, attention against float64 over the values the cache holds, and what the entry points refuse."""
import math

import pytest
import torch

from xotorch_support_jetson_amd.ops import kernels as K
from xotorch_support_jetson_amd.ops import reference as ref
from xotorch_support_jetson_amd.ops.rope import build_cos_sin

FMTS = ("mxfp4", "mxfp8")
PAGE = 64


# ------------------------------------------------------------------ oracles
def levels(fmt):
  if fmt == "mxfp4":
    return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
  return torch.tensor([(1 + c % 8 / 8) * 2.0 ** (c // 8 - 7) if c >= 8 else c / 8 * 2.0 ** -6 for c in range(127)], dtype=torch.float64)


def held(x, fmt):
  """The values that rows [..., Dh] of any type have in the cache, float64: the exponent by trying them all, elements by search."""
  lv, top, high = levels(fmt), {"mxfp4": 7.0, "mxfp8": 464.0}[fmt], {"mxfp4": 125, "mxfp8": 119}[fmt]
  g = x.double().cpu().unflatten(-1, (-1, 32))
  a = g.abs().amax(-1, keepdim=True)
  bad = ~torch.isfinite(a)
  steps = torch.arange(-100, high + 1, dtype=torch.float64)
  fits = torch.where(bad, 0.0, a) <= top * torch.exp2(steps)
  e = torch.where(fits.any(-1, keepdim=True), fits.int().argmax(-1, keepdim=True) - 100, high).double()
  y = (torch.where(bad, 0.0, g.abs()) / torch.exp2(e)).clamp(max=float(lv[-1]))
  up = torch.searchsorted(lv, y.contiguous()).clamp(max=len(lv) - 1)
  dn = (up - 1).clamp(min=0)
  lower = (y - lv[dn] < lv[up] - y) | ((y - lv[dn] == lv[up] - y) & (dn % 2 == 0))
  v = lv[torch.where(lower, dn, up)] * torch.exp2(e) * torch.sign(torch.where(bad, 1.0, g))
  return torch.where(bad, float("nan"), v).flatten(-2)


def pools(fmt, pages, Hkv, Dh, dev="cpu", fill=0):
  n = K.mx_page_bytes(fmt, Dh)
  return tuple(torch.full((pages, Hkv, n), fill, dtype=torch.uint8, device=dev) for _ in range(2))


def attend64(q, k, v, scale, past):
  """Causal attention in float64: q [n, H, Dh] at the end of k, v [past + n, Hkv, Dh]; also sum p |v| (rounding p moves the result by
  a share of it) and sum |q k|."""
  q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
  G = q.shape[1] // k.shape[1]
  k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
  s = torch.einsum("qhd,khd->hqk", q, k) * scale
  mag = torch.einsum("qhd,khd->hqk", q.abs(), k.abs()).amax(-1) * scale
  see = torch.arange(k.shape[0])[None] <= past + torch.arange(q.shape[0])[:, None]
  p = torch.softmax(s.masked_fill(~see, float("-inf")), -1)
  v = torch.where(see.any(0)[:, None, None], v, 0.0)
  return torch.einsum("hqk,khd->qhd", p, v), torch.einsum("hqk,khd->qhd", p, v.abs()), mag.t()[..., None]


def close(got, want, weight, mag):
  """Per element: the result's rounding to bf16 (2^-8 of it), the probabilities' (2^-8 each, so 2^-8 of sum p |v|), and the scores'
  error: products of 128 terms added in 32 bits (2^-17 of sum |q k|), the queries' split (2^-21 of the largest times sum |k|, within
  128 2^-21 <= 2^-14 of sum |q k| only where few dims carry it all: 2^-16 is taken for both), which moves p by twice that share."""
  got = got.double().cpu()
  tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -15 * mag) * weight + 1e-30
  assert torch.isfinite(got).all()
  worst = ((got - want).abs() / tol).max().item()
  assert worst <= 1.0, f"{worst} times the bound"


class Seqs:
  """Sequences of unlike length with pages in any order, and their cached values."""

  def __init__(self, fmt, ctx, Hkv, Dh, seed=0, dev="cpu", width=None, spare=2):
    g = torch.Generator().manual_seed(seed)
    pages = [-(-c // PAGE) for c in ctx]
    W = width or max(1, max(pages))
    pool = sum(pages) + spare
    self.tables = torch.zeros(len(ctx), W, dtype=torch.int32)
    order = torch.randperm(pool, generator=g).tolist()
    for b, n in enumerate(pages):
      for w in range(n):
        self.tables[b, w] = order.pop()
    self.ctx, self.lens, self.fmt, self.Dh = torch.tensor(ctx, dtype=torch.int32), ctx, fmt, Dh
    self.k, self.v = pools(fmt, pool, Hkv, Dh)
    chan = torch.exp(0.5 * torch.randn(Hkv, Dh, generator=g))
    self.kv = []
    for b, n in enumerate(ctx):
      k, v = torch.randn(n, Hkv, Dh, generator=g) * chan, torch.randn(n, Hkv, Dh, generator=g)
      t = torch.arange(n)
      ref.mx_write(k, v, self.tables[b].long()[t // PAGE] * PAGE + t % PAGE, self.k, self.v)
      self.kv.append((held(k, fmt), held(v, fmt)))
    self.to(dev)

  def to(self, dev):
    self.tables, self.ctx, self.k, self.v = (t.to(dev) for t in (self.tables, self.ctx, self.k, self.v))

  def spoil(self):
    """Every byte of the pools that holds no cached key becomes 0xff: NaN elements, and scales that read as NaN."""
    dev = self.k.device
    keep = ref.mx_read(self.k.cpu(), self.v.cpu(), torch.arange(self.k.shape[0]), self.Dh)
    self.k, self.v = torch.full_like(self.k, 255).cpu(), torch.full_like(self.v, 255).cpu()
    for b, n in enumerate(self.lens):
      t = torch.arange(n)
      at = self.tables[b].cpu().long()[t // PAGE], t % PAGE
      ref.mx_write(keep[0][at[0], :, at[1]], keep[1][at[0], :, at[1]], at[0] * PAGE + at[1], self.k, self.v)
    self.to(dev)


def check_decode(s, H, scale, seed=1, **kw):
  g = torch.Generator().manual_seed(seed)
  q = (2 * torch.randn(len(s.lens), H, s.Dh, generator=g)).to(torch.bfloat16)
  out = K.attn_decode_mx(q.to(s.k.device), s.k, s.v, s.tables, s.ctx, scale, **kw)
  for b, n in enumerate(s.lens):
    n = min(n, s.tables.shape[1] * PAGE)
    if n <= 0:
      assert (out[b] == 0).all()
      continue
    close(out[b:b + 1], *attend64(q[b:b + 1], s.kv[b][0][:n], s.kv[b][1][:n], scale, n - 1))
  return out


def check_prompt(s, new, H, scale, seed=1):
  g = torch.Generator().manual_seed(seed)
  cu = [0]
  for n in new:
    cu.append(cu[-1] + n)
  q = (2 * torch.randn(cu[-1] + 3, H, s.Dh, generator=g)).to(torch.bfloat16)
  dev = s.k.device
  out = torch.full((cu[-1] + 3, H, s.Dh), 7.0, dtype=torch.bfloat16, device=dev)
  K.attn_prefill_mx(q.to(dev), s.k, s.v, s.tables, torch.tensor(cu, dtype=torch.int32, device=dev), s.ctx, max(new), scale, out=out)
  for b, n in enumerate(new):
    if n:
      close(out[cu[b]:cu[b + 1]], *attend64(q[cu[b]:cu[b + 1]], *s.kv[b], scale, s.lens[b] - n))
  return out, cu[-1]


def qkv_of(T, H, Hkv, Dh, seed=0):
  g = torch.Generator().manual_seed(seed)
  return torch.randn(T, (H + 2 * Hkv) * Dh, generator=g).mul(torch.exp(torch.randn(T, 1, generator=g))).to(torch.bfloat16)


def rotated(x, pos, cs):
  """fp32 rotation, each product and sum rounded by itself."""
  c, s = cs[pos.long()][:, None].chunk(2, -1)
  a, b = x.float().chunk(2, -1)
  return torch.cat([a * c - b * s, b * c + a * s], -1)


# ------------------------------------------------------------------ format
@pytest.mark.parametrize("fmt", FMTS)
def test_format(fmt):
  g = torch.Generator().manual_seed(0)
  lv, top = levels(fmt), {"mxfp4": 7.0, "mxfp8": 464.0}[fmt]
  x = torch.randn(400, 32, generator=g) * torch.exp2(torch.randint(-130, 125, (400, 1), generator=g).float())
  ties = torch.cat([(lv[:-1] + lv[1:]) / 2, lv]).float()  # with the largest element beside them, so that the exponent is 0
  rows = [torch.cat([t, lv[-1:].float(), torch.zeros(31 - t.numel())]) * s for t in ties.split(31) for s in (1.0, -1.0, 2.0 ** 40)]
  rows += [torch.cat([torch.tensor([v]), torch.ones(31)]) for v in (top, math.nextafter(top, 1e9) * (1 + 2e-7), -top, top * 2.0 ** -90)]
  rows += [torch.zeros(32), torch.full((32,), 3e38), torch.full((32,), 1e-33), torch.full((32,), 2.0 ** -100)]
  x = torch.cat([x, torch.stack(rows)])
  code, scale = ref.mx_encode(x, fmt)
  assert torch.equal(ref.mx_decode(code, scale, fmt).double(), held(x, fmt))
  v = ref.mx_decode(code, scale, fmt)
  assert torch.equal(v, v.to(torch.bfloat16).float())  # what the cache holds is exact in bf16
  assert torch.equal(ref.mx_decode(*ref.mx_encode(v, fmt), fmt), v)


@pytest.mark.parametrize("fmt", FMTS)
def test_format_not_finite(fmt):
  x = torch.ones(4, 64)
  x[0, 3], x[1, 40], x[2, 63] = float("nan"), float("inf"), float("-inf")
  v = ref.mx_decode(*ref.mx_encode(x, fmt), fmt)
  assert torch.isnan(v[0, :32]).all() and torch.isnan(v[1, 32:]).all() and torch.isnan(v[2, 32:]).all()
  assert (v[0, 32:] == 1).all() and (v[1, :32] == 1).all() and (v[3] == 1).all()


@pytest.mark.parametrize("fmt,Dh,Hkv", [("mxfp4", 128, 2), ("mxfp8", 64, 3)])
def test_write_read(fmt, Dh, Hkv):
  check_write(fmt, Dh, 4, Hkv, 150, "cpu")


def check_write(fmt, Dh, H, Hkv, T, dev, seed=0):
  """Tokens to pages in any order, some to none: the pools' values against the search, other keys' bytes untouched."""
  g = torch.Generator().manual_seed(seed)
  pool = T // PAGE + 3
  slots = torch.randperm(pool * PAGE, generator=g)[:T]
  slots[::7] = -1
  slots[3::11] = pool * PAGE + 5
  x, pos, cs = qkv_of(T, H, Hkv, Dh, seed), torch.randint(0, 5000, (T,), generator=g, dtype=torch.int32), build_cos_sin(Dh, 5000, 10000.0)
  if T > 3:
    pos[1], pos[2] = -4, 9999  # (rows outside the table: its first and last)
  inside = pos.clamp(0, 4999)
  rows = x.view(T, H + 2 * Hkv, Dh)
  k, v = pools(fmt, pool, Hkv, Dh, fill=37)
  before = ref.mx_read(k, v, torch.arange(pool), Dh)
  kd, vd = k.to(dev), v.to(dev)
  on_cpu = dev == "cpu"
  q = K.rope_kv_write_mx(x.to(dev), (inside if on_cpu else pos).to(dev), cs.to(dev), slots.to(dev), kd, vd, H, Hkv)
  want_q = rotated(rows[:, :H], inside, cs)
  assert (q.cpu().float() - want_q).abs().le(2.0 ** -8 * want_q.abs() + 1e-30).all()
  got = ref.mx_read(kd.cpu(), vd.cpu(), torch.arange(pool), Dh)
  want_k, want_v = held(rotated(rows[:, H:H + Hkv], inside, cs), fmt), held(rows[:, H + Hkv:], fmt)
  fresh = torch.zeros(pool * PAGE, dtype=torch.bool)
  for t, s in enumerate(slots.tolist()):
    if 0 <= s < pool * PAGE:
      fresh[s] = True
      assert torch.equal(got[0][s // PAGE, :, s % PAGE].double(), want_k[t]), t
      assert torch.equal(got[1][s // PAGE, :, s % PAGE].double(), want_v[t]), t
  for a, b in zip(got, before):
    old = ~fresh.view(pool, 1, PAGE, 1).expand_as(a)
    assert torch.equal(a[old].nan_to_num(-1.0), b[old].nan_to_num(-1.0))
  # read back through tables: exact, zeros past the contexts, bad entries kept inside the pool
  tables = torch.tensor([[1, 0], [pool - 1, -3], [pool + 7, 2]], dtype=torch.int32)
  ctx = torch.tensor([100, 64, 1], dtype=torch.int32)
  kb, vb = K.kv_read_mx(kd, vd, tables.to(dev), ctx.to(dev), Dh)
  vb = ref.v_chunks(vb.cpu()).transpose(3, 4).flatten(2, 3)
  for b in range(3):
    for w in range(2):
      n = max(0, min(PAGE, int(ctx[b]) - w * PAGE))
      for out, src in ((kb.cpu(), got[0]), (vb, got[1])):
        page = out[2 * b + w].float()
        assert torch.equal(page[:, :n].nan_to_num(-1.0), src[min(max(int(tables[b, w]), 0), pool - 1)][:, :n].nan_to_num(-1.0))
        assert (page[:, n:] == 0).all()


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("fmt,Dh", [("mxfp4", 128), ("mxfp8", 64)])
def test_attention_cpu(fmt, Dh):
  s = Seqs(fmt, [70, 0, 1, 128], 2, Dh, width=3)
  check_decode(s, 4, Dh ** -0.5)
  s = Seqs(fmt, [70, 5, 128], 2, Dh)
  out, end = check_prompt(s, [10, 5, 1], 4, Dh ** -0.5)


def test_formats_refused():
  with pytest.raises(ValueError, match="mxfp4"):
    K.mx_page_bytes("int4", 128)
  k, v = pools("mxfp4", 2, 1, 128)
  with pytest.raises(ValueError, match="heads of 64"):
    K.mx_format(k, 64)
  with pytest.raises(ValueError):
    K.mx_format(k.to(torch.int8), 128)
  with pytest.raises(ValueError):
    ref.mx_format(torch.zeros(2, 1, K.mx_page_bytes("mxfp8", 32), dtype=torch.uint8), 32)


# ------------------------------------------------------------------ kernels
@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 64, 333, 2100])
@pytest.mark.parametrize("fmt,Dh,H,Hkv", [("mxfp4", 128, 4, 2), ("mxfp4", 64, 6, 3), ("mxfp8", 128, 7, 1), ("mxfp8", 64, 4, 4)])
def test_write_read_gpu(gpu, fmt, Dh, H, Hkv, T):
  check_write(fmt, Dh, H, Hkv, T, gpu, seed=T)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,Dh,H,Hkv", [("mxfp4", 128, 21, 8), ("mxfp8", 64, 30, 4)])
def test_write_many_heads_gpu(gpu, fmt, Dh, H, Hkv):
  """Rows enough for several heads a wave, heads that are no whole groups of those (37, 38)."""
  T = (1 << 17) // (H + 2 * Hkv) + 3
  assert T * (H + 2 * Hkv) >= 1 << 17
  check_write(fmt, Dh, H, Hkv, T, gpu)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_write_format_gpu(gpu, fmt):
  """Ties, borders of the exponent, values that vanish, overflow and are not finite, written as values (no rotation)."""
  lv, top = levels(fmt), {"mxfp4": 7.0, "mxfp8": 464.0}[fmt]
  ties = torch.cat([(lv[:-1] + lv[1:]) / 2, lv, -lv]).float()
  rows = [torch.cat([t, lv[-1:].float(), torch.zeros(31 - t.numel())]) * s for t in ties.split(31) for s in (1.0, 2.0 ** 40, 2.0 ** -90)]
  rows += [torch.cat([torch.tensor([v]), torch.ones(31)]) for v in (top, top * (1 + 2.0 ** -7), -top, top * 2.0 ** -90)]
  rows += [torch.zeros(32), torch.full((32,), 3e38), torch.full((32,), -3e38), torch.full((32,), 1e-33), torch.full((32,), 2.0 ** -100)]
  for bad in (float("nan"), float("inf"), float("-inf")):
    rows.append(torch.cat([torch.ones(9), torch.tensor([bad]), torch.ones(22)]))
  while len(rows) % 4:
    rows.append(torch.ones(32))
  x = torch.stack(rows).to(torch.bfloat16).view(-1, 128)  # (what is no bf16 is rounded first)
  T = x.shape[0]
  k, v = pools(fmt, T // PAGE + 1, 1, 128, gpu)
  cs = torch.cat([torch.ones(1, 64), torch.zeros(1, 64)], 1)
  qkv = torch.cat([torch.zeros_like(x), x, x], 1)
  K.rope_kv_write_mx(qkv.to(gpu), torch.zeros(T, dtype=torch.int32, device=gpu), cs.to(gpu), torch.arange(T, device=gpu), k, v, 1, 1)
  got = ref.mx_read(k.cpu(), v.cpu(), torch.arange(k.shape[0]), 128)
  want = held(x, fmt)
  assert torch.equal(got[1].reshape(-1, 128)[:T].double().nan_to_num(-1.0), want.nan_to_num(-1.0))
  fine = torch.isfinite(x.float()).all(-1) & (x.float().abs() < 1e38).all(-1)  # (an infinity times a sine of 0 is NaN in the other half)
  assert torch.equal(got[0].reshape(-1, 128)[:T][fine].double(), want[fine])
  kb, vb = K.kv_read_mx(k, v, torch.arange(k.shape[0], dtype=torch.int32, device=gpu)[:, None], torch.full((k.shape[0],), PAGE, dtype=torch.int32, device=gpu), 128)
  assert torch.equal(kb.cpu().float().nan_to_num(-1.0), got[0].nan_to_num(-1.0))
  assert torch.equal(ref.v_chunks(vb.cpu()).transpose(3, 4).flatten(2, 3).float().nan_to_num(-1.0), got[1].nan_to_num(-1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("Dh,H,Hkv", [(128, 8, 1), (128, 32, 2), (64, 14, 2), (64, 3, 3), (128, 5, 1)])
def test_decode_gpu(gpu, fmt, Dh, H, Hkv):
  s = Seqs(fmt, [1, 63, 64, 65, 0, 300, 128, 700], Hkv, Dh, dev=gpu, width=12)
  check_decode(s, H, Dh ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,Dh", [("mxfp4", 128), ("mxfp8", 128), ("mxfp4", 64), ("mxfp8", 64)])
def test_decode_stale_bytes_gpu(gpu, fmt, Dh):
  """Bytes past the contexts (of earlier requests, of anything) never reach a result."""
  s = Seqs(fmt, [1, 63, 65, 7, 0, 130], 2, Dh, dev=gpu, width=4)
  a = check_decode(s, 4, Dh ** -0.5)
  s.spoil()
  assert torch.equal(a, check_decode(s, 4, Dh ** -0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("waves", [(1, False), (2, False), (4, False), (4, True)])
@pytest.mark.parametrize("fmt,Dh,H,Hkv", [("mxfp4", 128, 8, 1), ("mxfp8", 128, 32, 2), ("mxfp4", 64, 3, 3), ("mxfp8", 64, 14, 2)])
def test_decode_parts_gpu(gpu, fmt, Dh, H, Hkv, waves, monkeypatch):
  """Contexts in parts, shorter ones than others and some without any: merged in the launch, the same whoever comes last, tickets left at
  zero; one sequence's parts more than one round of the merge."""
  s = Seqs(fmt, [1, 63, 64, 65, 0, 300, 640, 1350], Hkv, Dh, dev=gpu, width=22)
  s.spoil()
  monkeypatch.setattr(K, "mx_decode_waves", lambda *a: waves)
  for least in (1, 2, 5):
    monkeypatch.setattr(K.MXDecodeWorkspace, "parts", staticmethod(lambda b, h, pages: (least, -(-pages // least))))
    ws = K.MXDecodeWorkspace(8, H, Hkv, Dh, 22 * PAGE, gpu)
    a = check_decode(s, H, Dh ** -0.5, ws=ws)
    for _ in range(3):
      assert torch.equal(a, check_decode(s, H, Dh ** -0.5, ws=ws))
    assert (ws.tickets == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("order", [1, 2])
@pytest.mark.parametrize("B", [1, 2, 9, 63, 64])
def test_decode_order_gpu(gpu, B, order, monkeypatch):
  """Whatever order the sequences are taken in, each gets its own result: lengths alike, all but one, some of them 0, the same as given."""
  g = torch.Generator().manual_seed(B)
  for lens in ([130] * B, [130] * (B - 1) + [500], torch.randint(0, 300, (B,), generator=g).tolist()):
    s = Seqs("mxfp4", lens, 1, 64, dev=gpu, width=8)
    monkeypatch.setattr(K, "mx_decode_order", lambda *a: 0)
    a = check_decode(s, 2, 0.125, ws=K.MXDecodeWorkspace(B, 2, 1, 64, 512, gpu)) if B <= 9 else None
    monkeypatch.setattr(K, "mx_decode_order", lambda *a: order)
    monkeypatch.setattr(K.MXDecodeWorkspace, "parts", staticmethod(lambda b, h, pages: (pages, 1)))
    b = check_decode(s, 2, 0.125, ws=K.MXDecodeWorkspace(B, 2, 1, 64, 512, gpu))
    assert a is None or torch.allclose(a.float(), b.float(), rtol=2.0 ** -6, atol=2.0 ** -6)


@pytest.mark.gpu
def test_decode_workspace_gpu(gpu):
  """Wider tables than the workspace was made for, fewer sequences, and the rule's own choice at many sizes."""
  s = Seqs("mxfp4", [70, 1200, 0], 2, 64, dev=gpu, width=40)
  for max_ctx in (64, 700, 40 * PAGE):
    check_decode(s, 4, 0.125, ws=K.MXDecodeWorkspace(5, 4, 2, 64, max_ctx, gpu))
  with pytest.raises(RuntimeError, match="workspace"):
    check_decode(s, 4, 0.125, ws=K.MXDecodeWorkspace(2, 4, 2, 64, 4096, gpu))


def test_decode_parts_rule():
  for batch in (1, 3, 16, 64, 200, 512):
    for Hkv in (1, 2, 8, 32):
      for pages in (1, 4, 11, 16, 17, 64, 129, 513, 4096):
        least, most = K.MXDecodeWorkspace.parts(batch, Hkv, pages)
        assert 1 <= most <= pages and least * most >= pages and least <= 128
        ws = K.MXDecodeWorkspace(batch, 16, Hkv, 64, min(pages, 64) * PAGE, "meta")
        for b in (1, batch):
          least, most = ws.partition(b, pages)
          assert least * most >= pages and (most == 1 or b * most <= ws.rows) and most <= pages


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_decode_not_finite_gpu(gpu, fmt):
  """A NaN in a group of keys makes its sequence's heads NaN; one in a group of values those 32 dims; no other sequence."""
  s = Seqs(fmt, [100, 100, 100], 2, 128, dev=gpu)
  slot = lambda b, t: int(s.tables[b, t // PAGE]) * PAGE + t % PAGE  # noqa: E731
  k, v = (t.cpu() for t in (s.k, s.v))
  x = torch.ones(1, 2, 128)
  kb, vb = x.clone(), x.clone()
  kb[0, 0, 5] = float("nan")
  vb[0, 1, 40] = float("inf")
  ref.mx_write(kb, x, torch.tensor([slot(0, 70)]), k, v)
  ref.mx_write(x, vb, torch.tensor([slot(1, 3)]), k, v)
  q = torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(gpu)
  out = K.attn_decode_mx(q, k.to(gpu), v.to(gpu), s.tables, s.ctx, 0.1).cpu()
  bad = torch.zeros(3, 8, 128, dtype=torch.bool)
  bad[0, :4] = True
  bad[1, 4:, 32:64] = True
  assert torch.equal(torch.isnan(out), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,Dh,H,Hkv", [("mxfp4", 128, 8, 2), ("mxfp8", 64, 6, 3)])
def test_decode_range_gpu(gpu, fmt, Dh, H, Hkv):
  """Large and tiny queries: the split keeps their bits (scores of one dominant dim and of tiny ones beside it)."""
  s = Seqs(fmt, [90, 33], Hkv, Dh, dev=gpu)
  g = torch.Generator().manual_seed(3)
  for mul in (2.0 ** -60, 2.0 ** 60):
    q = torch.randn(2, H, Dh, generator=g)
    q[:, :, ::5] *= 2.0 ** -7
    q = (q * mul).to(torch.bfloat16)
    scale = 1.0 / mul / 8
    out = K.attn_decode_mx(q.to(gpu), s.k, s.v, s.tables, s.ctx, scale)
    for b, n in enumerate(s.lens):
      close(out[b:b + 1], *attend64(q[b:b + 1], *s.kv[b], scale, n - 1))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,Dh,H,Hkv", [("mxfp4", 128, 8, 2), ("mxfp8", 128, 4, 4), ("mxfp4", 64, 4, 2), ("mxfp8", 64, 8, 1)])
def test_prompt_gpu(gpu, fmt, Dh, H, Hkv, monkeypatch):
  ctx, new = [70, 5, 300, 128, 64, 1], [10, 5, 260, 1, 64, 1]
  s = Seqs(fmt, ctx, Hkv, Dh, dev=gpu, width=6)
  s.spoil()
  for direct, tiles in ((True, False), (True, True), (False, False)):  # from the pools, and through bf16 pages
    monkeypatch.setattr(K, "mx_prompt_direct", lambda *a: direct)
    monkeypatch.setattr(K, "mx_prompt_tiles", lambda *a: tiles)
    whole, end = check_prompt(s, new, H, Dh ** -0.5)
    assert (whole[end:] == 7).all()
  for limit in (1, 2 * 6 * Hkv * PAGE * Dh * 4):  # a sequence, two sequences at a time
    monkeypatch.setattr(K, "MX_READ_BYTES", limit)
    assert torch.equal(check_prompt(s, new, H, Dh ** -0.5)[0], whole)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,Dh,H,Hkv", [("mxfp4", 128, 4, 1), ("mxfp8", 128, 16, 1), ("mxfp4", 64, 7, 1), ("mxfp8", 64, 2, 2), ("mxfp4", 128, 3, 3)])
def test_turns_gpu(gpu, fmt, Dh, H, Hkv, monkeypatch):
  """A few new tokens behind long contexts (in parts), none, a token alone, more tokens than keys would allow."""
  s = Seqs(fmt, [1500, 2200, 33, 64, 1, 700], Hkv, Dh, dev=gpu, width=36)
  s.spoil()
  new = [3, 17, 0, 5, 1, 16]
  a, end = check_prompt(s, new, H, Dh ** -0.5)
  assert (a[end:] == 7).all()
  for _ in range(3):
    assert torch.equal(a, check_prompt(s, new, H, Dh ** -0.5)[0])
  s = Seqs(fmt, [3, 0], Hkv, Dh, dev=gpu)  # (rows before the first key: zeros, as in attn_prefill)
  for direct in (True, False):
    monkeypatch.setattr(K, "mx_prompt_direct", lambda *a: direct)
    q = torch.randn(7, H, Dh, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    out = K.attn_prefill_mx(q.to(gpu), s.k, s.v, s.tables, torch.tensor([0, 5, 7], dtype=torch.int32, device=gpu), s.ctx, 5, Dh ** -0.5)
    close(out[2:5], *attend64(q[2:5], *s.kv[0], Dh ** -0.5, 0))
    assert (out[:2] == 0).all() and (out[5:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,Dh,H,Hkv", [("mxfp4", 128, 4, 1), ("mxfp8", 128, 16, 1), ("mxfp4", 64, 7, 1), ("mxfp8", 64, 3, 3)])
def test_prompts_in_lds_gpu(gpu, fmt, Dh, H, Hkv, monkeypatch):
  """The kernel of four units: one page to many, waves without rows or without keys, tokens before the first key, a replayed result."""
  monkeypatch.setattr(K, "mx_prompt_tiles", lambda *a: True)
  s = Seqs(fmt, [1000, 470, 33, 64, 1, 129, 200], Hkv, Dh, dev=gpu, width=16)  # (16: in one part)
  s.spoil()
  a, end = check_prompt(s, [1000, 17, 0, 64, 1, 129, 5], H, Dh ** -0.5)
  assert (a[end:] == 7).all()
  assert torch.equal(a, check_prompt(s, [1000, 17, 0, 64, 1, 129, 5], H, Dh ** -0.5)[0])
  s = Seqs(fmt, [3, 0, 100], Hkv, Dh, dev=gpu)
  q = torch.randn(210, H, Dh, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
  out = K.attn_prefill_mx(q.to(gpu), s.k, s.v, s.tables, torch.tensor([0, 5, 7, 210], dtype=torch.int32, device=gpu), s.ctx, 203, Dh ** -0.5)
  close(out[2:5], *attend64(q[2:5], *s.kv[0], Dh ** -0.5, 0))
  close(out[110:], *attend64(q[110:], *s.kv[2], Dh ** -0.5, 0))
  assert (out[:2] == 0).all() and (out[5:110] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,Dh", [("mxfp4", 128), ("mxfp8", 64)])
def test_rising_scores_gpu(gpu, fmt, Dh, monkeypatch):
  """Scores that rise along the context, slowly, fast, then fall: weights against a maximum that is behind."""
  H, Hkv, n = 4, 2, 700
  s = Seqs(fmt, [n, 333], Hkv, Dh, dev=gpu)
  c = torch.randint(0, 2, (Dh,), generator=torch.Generator().manual_seed(0)) * 2.0 - 1
  t = torch.arange(n).float()
  rise = torch.where(t < 400, t / 100, torch.where(t < 600, 4 + (t - 400) / 8, 29 - (t - 600) / 16))  # scores in powers of e, at q = c
  s.kv = []
  for b, m in enumerate(s.lens):
    v = torch.randn(m, Hkv, Dh, generator=torch.Generator().manual_seed(b))
    k = (rise[:m, None, None] * c).expand(m, Hkv, Dh)
    at = s.tables[b].cpu().long()[torch.arange(m) // PAGE] * PAGE + torch.arange(m) % PAGE
    kc, vc = s.k.cpu(), s.v.cpu()
    ref.mx_write(k, v, at, kc, vc)
    s.k, s.v = kc.to(gpu), vc.to(gpu)
    s.kv.append((held(k, fmt), held(v, fmt)))
  q = (c + 0.05 * torch.randn(n + 333, H, Dh, generator=torch.Generator().manual_seed(9))).to(torch.bfloat16)
  out = K.attn_decode_mx(q[:2].to(gpu), s.k, s.v, s.tables, s.ctx, 1 / Dh)
  for b, m in enumerate(s.lens):
    close(out[b:b + 1], *attend64(q[b:b + 1], *s.kv[b], 1 / Dh, m - 1))
  for tiles in (True, False):
    monkeypatch.setattr(K, "mx_prompt_tiles", lambda *a: tiles)
    out = K.attn_prefill_mx(q.to(gpu), s.k, s.v, s.tables, torch.tensor([0, n, n + 333], dtype=torch.int32, device=gpu), s.ctx, n, 1 / Dh)
    for a, m, kv in ((0, n, s.kv[0]), (n, 333, s.kv[1])):
      close(out[a:a + m], *attend64(q[a:a + m], *kv, 1 / Dh, 0))


@pytest.mark.gpu
def test_prompts_of_many_sequences_gpu(gpu):
  """More sequences than a grid dimension holds: few unlike ones over and over."""
  s = Seqs("mxfp4", [70, 1, 64, 130, 0], 1, 64, dev=gpu)
  n, H = 14000, 2
  q = torch.randn(5, H, 64, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
  cu = torch.arange(5 * n + 1, dtype=torch.int32, device=gpu)
  out = K.attn_prefill_mx(q.to(gpu).repeat(n, 1, 1), s.k, s.v, s.tables.repeat(n, 1), cu, s.ctx.repeat(n), 1, 0.125).view(n, 5, H, 64)
  assert (out == out[:1]).all() and (out[0, 4] == 0).all()
  for b in range(4):
    close(out[0, b:b + 1], *attend64(q[b:b + 1], *s.kv[b], 0.125, s.lens[b] - 1))


@pytest.mark.gpu
@pytest.mark.parametrize("B", [6, 63, 64, 65, 130, 4200])
def test_steps_of_unlike_lengths_gpu(gpu, B):
  """One long prompt among short turns, single tokens and sequences without any: every unit finds its sequence."""
  H, Hkv, Dh = 6, 2, 64
  s = Seqs("mxfp4", [70, 33, 130, 5, 64, 800], Hkv, Dh, dev=gpu)
  new = [1, 0, 21, 5, 1, 790]
  g = torch.Generator().manual_seed(B)
  qs = [torch.randn(n, H, Dh, generator=g).to(torch.bfloat16) for n in new]
  which = [i % 5 for i in range(B)]
  which[B // 2] = 5
  cu = [0]
  for i in which:
    cu.append(cu[-1] + new[i])
  q = torch.cat([qs[i] for i in which]).to(gpu)
  at = torch.tensor(which, device=gpu)
  out = K.attn_prefill_mx(q, s.k, s.v, s.tables[at], torch.tensor(cu, dtype=torch.int32, device=gpu), s.ctx[at], 790, 0.125).cpu()
  first = {}
  for b, i in enumerate(which):
    o = out[cu[b]:cu[b + 1]]
    if i not in first:
      first[i] = o
      if new[i]:
        close(o, *attend64(qs[i], *s.kv[i], 0.125, s.lens[i] - new[i]))
    else:
      assert torch.equal(o, first[i]), b


@pytest.mark.gpu
@pytest.mark.parametrize("cu", [[0, 30, 20, 40], [5, 5, 900, 3], [-7, 2, 3, 1 << 30], [40, 30, 20, 10]])
def test_starts_that_fall_gpu(gpu, cu):
  """Starts that are not in order (nothing a caller should give) read and write within the tensors, whatever they give."""
  s = Seqs("mxfp4", [70, 33, 130], 2, 64, dev=gpu)
  q = torch.randn(40, 4, 64, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(gpu)
  whole = torch.full((80, 4, 64), 7.0, dtype=torch.bfloat16, device=gpu)
  for most in (40, 400):
    K.attn_prefill_mx(q, s.k, s.v, s.tables, torch.tensor(cu, dtype=torch.int32, device=gpu), s.ctx, most, 0.125, out=whole[20:60])
    assert (whole[:20] == 7).all() and (whole[60:] == 7).all()


@pytest.mark.gpu
def test_far_pages_gpu(gpu):
  """Pages whose bytes lie past 2^32 of their pool: written, read back, attended to by single tokens and prompts."""
  Hkv, Dh, fmt = 8, 128, "mxfp8"
  pool = (1 << 32) // (Hkv * K.mx_page_bytes(fmt, Dh)) + 9
  k, v = (torch.empty(pool, Hkv, K.mx_page_bytes(fmt, Dh), dtype=torch.uint8, device=gpu) for _ in range(2))
  T, H = 70, 16
  x, cs = qkv_of(T, H, Hkv, Dh), build_cos_sin(Dh, T, 10000.0)
  pages = torch.tensor([pool - 1, pool - 4])
  t = torch.arange(T)
  slots = pages[t // PAGE] * PAGE + t % PAGE
  q = K.rope_kv_write_mx(x.to(gpu), t.int().to(gpu), cs.to(gpu), slots.to(gpu), k, v, H, Hkv)
  rows = x.view(T, H + 2 * Hkv, Dh)
  kw, vw = held(rotated(rows[:, H:H + Hkv], t, cs), fmt), held(rows[:, H + Hkv:], fmt)
  tables, ctx = pages.int()[None].to(gpu), torch.tensor([T], dtype=torch.int32, device=gpu)
  kb, vb = K.kv_read_mx(k, v, tables, ctx, Dh)
  assert torch.equal(kb.cpu().transpose(1, 2).flatten(0, 1)[:T].double(), kw)
  assert torch.equal(ref.v_chunks(vb.cpu()).transpose(3, 4).flatten(2, 3).transpose(1, 2).flatten(0, 1)[:T].double(), vw)
  qc = q.cpu()
  close(K.attn_decode_mx(q[-1:], k, v, tables, ctx, 0.1), *attend64(qc[-1:], kw, vw, 0.1, T - 1))
  close(K.attn_prefill_mx(q[-9:].contiguous(), k, v, tables, torch.tensor([0, 9], dtype=torch.int32, device=gpu), ctx, 9, 0.1),
        *attend64(qc[-9:], kw, vw, 0.1, T - 9))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,Dh", [("mxfp4", 128), ("mxfp8", 64)])
def test_captured_steps_gpu(gpu, fmt, Dh):
  """A decode step (write, attention in parts) and a prompt's attention in one graph, replayed with new inputs between eager work of the
  same kind, on a stream of its own; every replay against eager calls."""
  H, Hkv, B = 8, 2, 3
  s = Seqs(fmt, [300, 70, 900], Hkv, Dh, dev=gpu, width=16)
  cs = build_cos_sin(Dh, 1024, 10000.0).to(gpu)
  g = torch.Generator().manual_seed(0)
  pos = s.ctx - 1
  slots = (s.tables.gather(1, (pos // PAGE).long()[:, None])[:, 0].long() * PAGE + pos % PAGE)
  x = torch.zeros(B, (H + 2 * Hkv) * Dh, dtype=torch.bfloat16, device=gpu)
  qp = torch.zeros(12, H, Dh, dtype=torch.bfloat16, device=gpu)
  cu = torch.tensor([0, 5, 6, 12], dtype=torch.int32, device=gpu)
  ws = K.MXDecodeWorkspace(B, H, Hkv, Dh, 1024, gpu)
  assert ws.partition(B, 16)[1] > 1

  def step(ws):
    q = K.rope_kv_write_mx(x, pos, cs, slots, s.k, s.v, H, Hkv)
    return K.attn_decode_mx(q, s.k, s.v, s.tables, s.ctx, 0.1, ws), K.attn_prefill_mx(qp, s.k, s.v, s.tables, cu, s.ctx, 6, 0.1)
  stream = torch.cuda.Stream(gpu)
  stream.wait_stream(torch.cuda.current_stream(gpu))
  with torch.cuda.stream(stream):
    step(ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
      outs = step(ws)
  torch.cuda.synchronize()
  for i in range(5):
    x.copy_(qkv_of(B, H, Hkv, Dh, i).to(gpu))
    qp.copy_(torch.randn(qp.shape, generator=g).to(torch.bfloat16))
    graph.replay()
    got = [t.clone() for t in outs]
    torch.cuda.synchronize()
    for a, b in zip(got, step(K.MXDecodeWorkspace(B, H, Hkv, Dh, 1024, gpu))):
      assert torch.equal(a, b), i


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_queries_not_finite_gpu(gpu, fmt):
  """A query that is not finite makes its own row NaN and no other; zeros weigh all keys alike."""
  s = Seqs(fmt, [100, 33], 2, 128, dev=gpu)
  q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
  q[0, 1, 7], q[1, 6, 100], q[1, 2] = float("nan"), float("inf"), 0.0
  out = K.attn_decode_mx(q.to(gpu), s.k, s.v, s.tables, s.ctx, 0.1).cpu()
  bad = torch.zeros(2, 8, dtype=torch.bool)
  bad[0, 1] = bad[1, 6] = True
  assert torch.equal(torch.isnan(out).any(-1), bad) and torch.isnan(out[bad]).all()
  assert torch.allclose(out[1, 2].double(), s.kv[1][1][:, 0].mean(0), rtol=2.0 ** -7, atol=2.0 ** -7)
  cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu)
  out = K.attn_prefill_mx(q.to(gpu), s.k, s.v, s.tables, cu, s.ctx, 1, 0.1).cpu()
  assert torch.equal(torch.isnan(out).any(-1), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,Dh", [("mxfp4", 128), ("mxfp8", 64)])
def test_outputs_given_gpu(gpu, fmt, Dh):
  """Results into the caller's tensors, the attentions' into their queries too; pages read back into used ones, with and without the tables'
  rest."""
  H, Hkv = 8, 2
  s = Seqs(fmt, [70, 1200, 5], Hkv, Dh, dev=gpu, width=24)
  g = torch.Generator().manual_seed(0)
  x, pos, cs = qkv_of(9, H, Hkv, Dh).to(gpu), torch.arange(9, dtype=torch.int32, device=gpu), build_cos_sin(Dh, 16, 10000.0).to(gpu)
  none = torch.full((9,), -1, device=gpu)
  want = K.rope_kv_write_mx(x, pos, cs, none, s.k, s.v, H, Hkv)
  flat = torch.empty(9, H * Dh, dtype=torch.bfloat16, device=gpu)
  assert K.rope_kv_write_mx(x, pos, cs, none, s.k, s.v, H, Hkv, q_out=flat).data_ptr() == flat.data_ptr() and torch.equal(flat.view_as(want), want)
  q = torch.randn(3, H, Dh, generator=g).to(torch.bfloat16).to(gpu)
  want = K.attn_decode_mx(q, s.k, s.v, s.tables, s.ctx, 0.1)
  assert torch.equal(K.attn_decode_mx(q, s.k, s.v, s.tables, s.ctx, 0.1, out=q), want) and torch.equal(q, want)
  cu = torch.tensor([0, 40, 46, 49], dtype=torch.int32, device=gpu)
  for most in (40, 1500):  # (the second: a bound only)
    q = torch.randn(49, H, Dh, generator=g).to(torch.bfloat16).to(gpu)
    want = K.attn_prefill_mx(q, s.k, s.v, s.tables, cu, s.ctx, most, 0.1)
    assert torch.equal(K.attn_prefill_mx(q, s.k, s.v, s.tables, cu, s.ctx, most, 0.1, out=q), want) and torch.equal(q, want)
  k, v = K.kv_read_mx(s.k, s.v, s.tables, s.ctx, Dh)
  for skip in (False, True):
    ko, vo = torch.full_like(k, 3.0), torch.full_like(v, 3.0)
    K.kv_read_mx(s.k, s.v, s.tables, s.ctx, Dh, ko, vo, skip)
    past = (torch.arange(24, device=gpu)[None] * PAGE >= s.ctx[:, None]).flatten()
    for a, b in ((ko, k), (vo, v)):
      assert torch.equal(a[~past], b[~past]) and (a[past] == (3.0 if skip else 0.0)).all()


@pytest.mark.gpu
def test_two_streams_gpu(gpu):
  """Calls in flight on two streams at once, single tokens with a workspace each."""
  H, Hkv, Dh = 8, 2, 128
  s = Seqs("mxfp4", [4000, 1200, 900], Hkv, Dh, dev=gpu)
  cu = torch.tensor([0, 9, 12, 20], dtype=torch.int32, device=gpu)
  qs = [torch.randn(20, H, Dh, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).to(gpu) for i in range(2)]
  ws = [K.MXDecodeWorkspace(3, H, Hkv, Dh, 4096, gpu) for _ in range(2)]

  def both(i):
    return K.attn_decode_mx(qs[i][:3], s.k, s.v, s.tables, s.ctx, 0.1, ws[i]), K.attn_prefill_mx(qs[i], s.k, s.v, s.tables, cu, s.ctx, 9, 0.1)
  want = [both(i) for i in range(2)]
  streams = [torch.cuda.Stream(gpu) for _ in range(2)]
  torch.cuda.synchronize()
  got = []
  for n in range(10):
    for i, stream in enumerate(streams):
      with torch.cuda.stream(stream):
        got.append((i, both(i)))
  torch.cuda.synchronize()
  for i, (a, b) in got:
    assert torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])


@pytest.mark.gpu
def test_nothing_to_do_gpu(gpu):
  s = Seqs("mxfp4", [70, 5], 2, 128, dev=gpu)
  none = lambda *shape, dt=torch.bfloat16: torch.zeros(*shape, dtype=dt, device=gpu)  # noqa: E731
  assert K.attn_decode_mx(none(0, 4, 128), s.k, s.v, none(0, 3, dt=torch.int32), none(0, dt=torch.int32), 1.0).shape == (0, 4, 128)
  assert K.rope_kv_write_mx(none(0, 8 * 128), none(0, dt=torch.int32), none(9, 128, dt=torch.float32), none(0, dt=torch.int64), s.k, s.v, 4, 2).shape == (0, 4, 128)
  assert K.kv_read_mx(s.k, s.v, none(0, 3, dt=torch.int32), none(0, dt=torch.int32), 128)[0].shape == (0, 2, 64, 128)
  out = torch.ones(3, 4, 128, dtype=torch.bfloat16, device=gpu)
  K.attn_prefill_mx(none(3, 4, 128), s.k, s.v, s.tables, none(3, dt=torch.int32), s.ctx, 0, 1.0, out=out)
  assert (out == 1).all()


@pytest.mark.gpu
def test_refusals_gpu(gpu):
  s = Seqs("mxfp4", [70, 5], 2, 128, dev=gpu)
  q = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device=gpu)
  bad = [
    lambda: K.attn_decode_mx(q.float(), s.k, s.v, s.tables, s.ctx, 1.0),
    lambda: K.attn_decode_mx(q, s.k.to(torch.int8), s.v, s.tables, s.ctx, 1.0),
    lambda: K.attn_decode_mx(q, s.k, s.v[..., :-64].contiguous(), s.tables, s.ctx, 1.0),
    lambda: K.attn_decode_mx(q[..., :64].contiguous(), s.k, s.v, s.tables, s.ctx, 1.0),
    lambda: K.attn_decode_mx(q, s.k, s.v, s.tables.long(), s.ctx, 1.0),
    lambda: K.attn_decode_mx(q, s.k, s.v, s.tables[:1], s.ctx, 1.0),
    lambda: K.attn_decode_mx(q, s.k, s.v, s.tables, s.ctx[:1], 1.0),
    lambda: K.attn_decode_mx(q, s.k.cpu(), s.v, s.tables, s.ctx, 1.0),
    lambda: K.attn_decode_mx(q[:, :3].contiguous(), s.k, s.v, s.tables, s.ctx, 1.0),
    lambda: K.attn_decode_mx(torch.zeros(2, 34, 128, dtype=torch.bfloat16, device=gpu), s.k, s.v, s.tables, s.ctx, 1.0),
    lambda: K.attn_decode_mx(q, s.k, s.v, s.tables, s.ctx, 0.0),
    lambda: K.attn_decode_mx(q, s.k, s.v, s.tables, s.ctx, float("nan")),
    lambda: K.attn_decode_mx(q, s.k, s.v, s.tables, s.ctx, 1.0, out=q.float()),
    lambda: K.attn_prefill_mx(q, s.k, s.v, s.tables, torch.tensor([0, 2], dtype=torch.int32, device=gpu), s.ctx, 1, 1.0),
    lambda: K.attn_prefill_mx(q, s.k, s.v, s.tables, torch.tensor([0, 1, 2], device=gpu), s.ctx, 1, 1.0),
    lambda: K.kv_read_mx(s.k, s.v, s.tables, s.ctx[:1], 128),
    lambda: K.kv_read_mx(s.k, s.v, s.tables, s.ctx, 64),
    lambda: K.kv_read_mx(s.k, s.v, s.tables, s.ctx, 128, k_out=torch.zeros(1, 2, 64, 128, dtype=torch.bfloat16, device=gpu)),
    lambda: K.rope_kv_write_mx(torch.zeros(3, 6 * 128, dtype=torch.bfloat16, device=gpu), torch.zeros(2, dtype=torch.int32, device=gpu),
                               torch.zeros(9, 128, device=gpu), torch.zeros(3, dtype=torch.int64, device=gpu), s.k, s.v, 2, 2),
    lambda: K.rope_kv_write_mx(torch.zeros(3, 6 * 128, dtype=torch.bfloat16, device=gpu), torch.zeros(3, dtype=torch.int32, device=gpu),
                               torch.zeros(9, 128, device=gpu), torch.zeros(3, dtype=torch.int64, device=gpu), s.k, s.v, 4, 1),
    lambda: K.rope_kv_write_mx(torch.zeros(3, 6 * 128, dtype=torch.bfloat16, device=gpu), torch.zeros(3, dtype=torch.int32, device=gpu),
                               torch.zeros(9, 64, device=gpu), torch.zeros(3, dtype=torch.int64, device=gpu), s.k, s.v, 2, 2),
  ]
  for i, call in enumerate(bad):
    with pytest.raises((RuntimeError, ValueError)):
      call()
      print("not refused:", i)


# ------------------------------------------------------------------ edges
SCALES_REFUSED = (0.0, -1.0, 1e-50, 1e-38, 1e-310, 2e38, 3e38, 1e300, float("inf"), float("nan"))


def check_scales(dev):
  """A scale that vanishes or overflows as the float that scores are multiplied by; the bounds themselves pass."""
  s = Seqs("mxfp8", [70, 5], 2, 128, dev=dev)
  q = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device=dev)
  cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
  for scale in SCALES_REFUSED:
    with pytest.raises(RuntimeError, match="scale"):
      K.attn_decode_mx(q, s.k, s.v, s.tables, s.ctx, scale)
    with pytest.raises(RuntimeError, match="scale"):
      K.attn_prefill_mx(q, s.k, s.v, s.tables, cu, s.ctx, 1, scale)
  for scale in (2.0 ** -125, 2.0 ** 126):  # (queries of zeros: every key weighs alike)
    for out in (K.attn_decode_mx(q, s.k, s.v, s.tables, s.ctx, scale), K.attn_prefill_mx(q, s.k, s.v, s.tables, cu, s.ctx, 1, scale)):
      for b, n in enumerate(s.lens):
        close(out[b:b + 1], *attend64(q[b:b + 1], *s.kv[b], 1.0, n - 1))


def test_scales():
  check_scales("cpu")


@pytest.mark.gpu
def test_scales_gpu(gpu, monkeypatch):
  for direct in (True, False):
    monkeypatch.setattr(K, "mx_prompt_direct", lambda *a: direct)
    check_scales(gpu)
  s = Seqs("mxfp4", [70, 5], 2, 128, dev=gpu)
  q = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device=gpu)
  monkeypatch.setattr(K, "_mx_scale", lambda scale: None)  # (the binding by itself)
  for scale in SCALES_REFUSED:
    with pytest.raises(RuntimeError, match="scale"):
      K.attn_decode_mx(q, s.k, s.v, s.tables, s.ctx, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("far", [1e31, -1e31, 1e37, -1e37, 1e12, -1e12, 3e7])
@pytest.mark.parametrize("fmt,Dh", [("mxfp4", 128), ("mxfp8", 128), ("mxfp4", 64), ("mxfp8", 64)])
def test_far_scores_gpu(gpu, fmt, Dh, far, monkeypatch):
  """Scores of any finite size (of either sign, past the precision of their products): equal ones weigh alike, a largest one takes all.
  Every product is a power of two times 207 / 128 and 1, 1.5 or 0, so scores are exact and weights 1 or 0: the result is off by its rounding
  and its sum's, n <= 200 terms of 2^-24 each."""
  H, Hkv = 4, 2
  s = Seqs(fmt, [200, 130, 70], Hkv, Dh, dev=gpu)
  a = round(math.log2(abs(far) / Dh) / 2)
  c = torch.randint(0, 2, (Dh,), generator=torch.Generator().manual_seed(0)) * 2.0 - 1
  levels = [torch.ones(200), torch.where(torch.arange(130) % 7 == 3, 1.5, 1.0), torch.where(torch.arange(70) % 5 == 2, 0.0, 1.0)]
  s.kv = []
  for b, m in enumerate(s.lens):
    v = torch.randn(m, Hkv, Dh, generator=torch.Generator().manual_seed(b))
    k = (levels[b][:, None, None] * c * 2.0 ** a).expand(m, Hkv, Dh)
    at = s.tables[b].cpu().long()[torch.arange(m) // PAGE] * PAGE + torch.arange(m) % PAGE
    kc, vc = s.k.cpu(), s.v.cpu()
    ref.mx_write(k, v, at, kc, vc)
    s.k, s.v = kc.to(gpu), vc.to(gpu)
    s.kv.append((held(k, fmt), held(v, fmt)))
    assert torch.equal(s.kv[b][0], k.double())
  q = (c * 2.0 ** a * math.copysign(207 / 128, far)).expand(400, H, Dh).to(torch.bfloat16).contiguous()

  def check(out, rows, b, past):
    want, weight, _ = attend64(q[:rows], *s.kv[b], 0.9, past)
    assert ((out.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -16 * weight).all()
  for waves in ((1, False), (2, False), (4, True)):
    for least in (1, 4):
      with monkeypatch.context() as m:
        m.setattr(K, "mx_decode_waves", lambda *a: waves)
        m.setattr(K.MXDecodeWorkspace, "parts", staticmethod(lambda b, h, pages: (least, -(-pages // least))))
        out = K.attn_decode_mx(q[:3].contiguous().to(gpu), s.k, s.v, s.tables, s.ctx, 0.9)
      for b, n in enumerate(s.lens):
        check(out[b:b + 1], 1, b, n - 1)
  cu = [0, 200, 330, 400]
  for tiles in (True, False):
    monkeypatch.setattr(K, "mx_prompt_tiles", lambda *a: tiles)
    out = K.attn_prefill_mx(q.to(gpu), s.k, s.v, s.tables, torch.tensor(cu, dtype=torch.int32, device=gpu), s.ctx, 200, 0.9)
    for b, n in enumerate(s.lens):
      check(out[cu[b]:cu[b + 1]], n, b, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,Dh", [("mxfp4", 128), ("mxfp8", 128), ("mxfp4", 64), ("mxfp8", 64)])
def test_rows_without_keys_gpu(gpu, fmt, Dh, monkeypatch):
  """Tokens before the first key give zeros whatever the cache holds, NaN too; the others see it."""
  H, Hkv = 4, 2
  s = Seqs(fmt, [3, 70], Hkv, Dh, dev=gpu)
  k, v = s.k.cpu(), s.v.cpu()
  bad = torch.full((1, Hkv, Dh), float("nan"))
  for b in range(2):
    ref.mx_write(bad, bad, s.tables[b, :1].cpu().long() * PAGE, k, v)
  q = torch.randn(87, H, Dh, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(gpu)
  cu = torch.tensor([0, 7, 87], dtype=torch.int32, device=gpu)
  for tiles in (True, False):
    monkeypatch.setattr(K, "mx_prompt_tiles", lambda *a: tiles)
    out = K.attn_prefill_mx(q, k.to(gpu), v.to(gpu), s.tables, cu, s.ctx, 80, 0.1)
    assert (out[:4] == 0).all() and (out[7:17] == 0).all()
    assert torch.isnan(out[4:7]).all() and torch.isnan(out[17:]).all()


@pytest.mark.parametrize("fmt,Dh", [("mxfp4", 128), ("mxfp8", 64)])
def test_prompt_rows_cpu(fmt, Dh):
  """On the CPU as on the GPU: tokens before the first key give zeros, rows of no sequence stay, contexts end with their table, a NaN
  reaches the tokens that see it."""
  s = Seqs(fmt, [3, 0, 100, 70], 2, Dh)
  q = torch.randn(33, 4, Dh, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
  cu = torch.tensor([0, 5, 7, 7, 30], dtype=torch.int32)
  out = K.attn_prefill_mx(q, s.k, s.v, s.tables, cu, s.ctx, 23, 0.1, out=torch.full_like(q, 7.0))
  assert (out[:2] == 0).all() and (out[5:7] == 0).all() and (out[30:] == 7).all()
  close(out[2:5], *attend64(q[2:5], *s.kv[0], 0.1, 0))
  close(out[7:30], *attend64(q[7:30], *s.kv[3], 0.1, 47))
  n = s.tables.shape[1] * PAGE
  past = K.attn_prefill_mx(q[:1], s.k, s.v, s.tables[2:3], torch.tensor([0, 1], dtype=torch.int32), torch.tensor([n + 60], dtype=torch.int32), 1, 0.1)
  whole = K.attn_prefill_mx(q[:1], s.k, s.v, s.tables[2:3], torch.tensor([0, 1], dtype=torch.int32), torch.tensor([n], dtype=torch.int32), 1, 0.1)
  assert torch.equal(past, whole)
  bad = torch.ones(1, 2, Dh)
  bad[0, 1, 40] = float("nan")
  ref.mx_write(torch.ones(1, 2, Dh), bad, s.tables[3, 0:1].long() * PAGE + 50, s.k, s.v)
  got = K.attn_prefill_mx(q, s.k, s.v, s.tables, cu, s.ctx, 23, 0.1)[7:30]
  want = torch.zeros(23, 4, Dh, dtype=torch.bool)
  want[3:, 2:, 32:64] = True
  assert torch.equal(torch.isnan(got), want)


@pytest.mark.parametrize("fmt,Dh", [("mxfp4", 128), ("mxfp8", 64)])
def test_read_skips_cpu(fmt, Dh):
  """Pages read back into used ones: those wholly past a context become zeros, or (skip) stay, on the CPU too."""
  s = Seqs(fmt, [70, 0, 130], 2, Dh, width=4)
  k, v = K.kv_read_mx(s.k, s.v, s.tables, s.ctx, Dh)
  past = (torch.arange(4)[None] * PAGE >= s.ctx[:, None]).flatten()
  for skip in (False, True):
    ko, vo = torch.full_like(k, 3.0), torch.full_like(v, 3.0)
    K.kv_read_mx(s.k, s.v, s.tables, s.ctx, Dh, ko, vo, skip)
    for a, b in ((ko, k), (vo, v)):
      assert torch.equal(a[~past], b[~past]) and (a[past] == (3.0 if skip else 0.0)).all()


def test_prompt_form_by_contexts(monkeypatch):
  """Long portions of mxfp8 go over bf16 pages where their contexts are long, not where only the table is wide."""
  asked = []
  monkeypatch.setattr(K, "_gpu", lambda t: True)
  monkeypatch.setattr(K, "mx_prompt_direct", lambda rows, pages, *a, rule=K.mx_prompt_direct: asked.append((pages, rule(rows, pages, *a))) or True)

  class Bindings:
    def attn_prompt_mx(self, *a):
      asked.append(a[-4:-1])
  monkeypatch.setattr(K, "require", Bindings)
  k, v = pools("mxfp8", 2, 8, 128)
  q = torch.zeros(2048, 32, 128, dtype=torch.bfloat16)
  cu, tables = torch.tensor([0, 2048], dtype=torch.int32), torch.zeros(1, 2048, dtype=torch.int32)

  def ask(max_ctx, q=q):
    asked.clear()
    K.attn_prefill_mx(q, k, v, tables, cu, cu[1:], q.shape[0], 1.0, max_ctx=max_ctx)
    return asked[0]
  assert ask(2048) == (32, True) and ask(2049) == (33, True) and ask(16384) == (256, False) and ask(0) == (2048, False)
  assert ask(1 << 20) == (2048, False)  # (a bound past the table says no more than the table)
  ask(4000, q[:8])  # few rows: parts of such a context, not of the table
  pages_of_part, parts, _ = asked[1]
  assert parts == K.mx_prompt_parts(8, 63) > 1 and parts * pages_of_part >= 63


def test_decode_form_by_contexts(monkeypatch):
  """Parts, waves and order of single tokens by their longest context where it is known, in a table of any width."""
  asked = []

  class Bindings:
    def attn_decode_mx(self, *a):
      asked.append(a[9:14])
  monkeypatch.setattr(K, "_gpu", lambda t: True)
  monkeypatch.setattr(K, "require", Bindings)
  k, v = pools("mxfp8", 2, 8, 128)
  for B, n in ((1, 700), (4, 3000), (64, 5000), (512, 520), (300, 9000)):
    q, ctx = torch.zeros(B, 32, 128, dtype=torch.bfloat16), torch.full((B,), n, dtype=torch.int32)
    ws = K.MXDecodeWorkspace(B, 32, 8, 128, 2048 * PAGE, "meta")
    for width, bound in ((-(-n // PAGE), 0), (2048, n), (-(-n // PAGE), 1 << 20)):
      K.attn_decode_mx(q, k, v, torch.zeros(B, width, dtype=torch.int32), ctx, 1.0, ws, max_ctx=bound)
    assert asked[-3] == asked[-2] == asked[-1], asked[-3:]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_contexts_past_their_bound_gpu(gpu, fmt, monkeypatch):
  """A bound chooses the form and nothing else: results are right where contexts pass it too."""
  s = Seqs(fmt, [1500, 33, 0, 700], 2, 128, dev=gpu, width=40)
  for bound in (1, 64, 700, 1500, 1 << 20):
    check_decode(s, 8, 128 ** -0.5, max_ctx=bound)
    check_decode(s, 8, 128 ** -0.5, max_ctx=bound, ws=K.MXDecodeWorkspace(4, 8, 2, 128, 40 * PAGE, gpu))
  new = [5, 3, 0, 9]
  prefill = K.attn_prefill_mx
  for bound in (1, 700, 1500):
    monkeypatch.setattr(K, "attn_prefill_mx", lambda *a, **kw: prefill(*a, **kw, max_ctx=bound))
    check_prompt(s, new, 8, 128 ** -0.5)


def test_prompt_pages_in_bounds(monkeypatch):
  """Starts out of range reach the bf16 kernel, which takes them as they are, within the tokens; entries too few or too many are refused
  whatever the form."""
  import contextlib
  starts = []

  class Bindings:
    def kv_read_mx(self, *a):
      pass

    def attn_prefill(self, q, k, v, tables, cu, ctx, *a):
      starts.append((cu.tolist(), ctx.tolist(), cu.dtype, ctx.dtype))
  monkeypatch.setattr(K, "_gpu", lambda t: True)
  monkeypatch.setattr(K, "require", Bindings)
  monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
  monkeypatch.setattr(K, "mx_prompt_direct", lambda *a: False)
  k, v = pools("mxfp8", 2, 2, 128)
  q, tables = torch.zeros(40, 4, 128, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32)
  ctx = torch.tensor([70, -3, 130], dtype=torch.int32)
  for cu in ([0, 30, 20, 40], [5, 5, 900, 3], [-7, 2, 3, 1 << 30]):
    K.attn_prefill_mx(q, k, v, tables, torch.tensor(cu, dtype=torch.int32), ctx, 40, 1.0)
    got, lens, *types = starts.pop()
    assert got == [min(max(c, 0), 40) for c in cu] and lens == [70, 0, 130] and types == [torch.int32] * 2
  for direct in (True, False):
    monkeypatch.setattr(K, "mx_prompt_direct", lambda *a: direct)
    for n, m, most in ((4, 4, 40), (3, 3, 40), (5, 3, 40), (4, 2, 40), (4, 3, 1 << 24), (4, 3, -1)):
      with pytest.raises(RuntimeError, match="attn_prefill_mx"):
        K.attn_prefill_mx(q, k, v, tables, torch.zeros(n, dtype=torch.int32), torch.ones(m, dtype=torch.int32), most, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("cu", [[0, 30, 20, 40], [5, 5, 900, 3], [-7, 2, 3, 1 << 30], [40, 30, 20, 10]])
def test_starts_that_fall_pages_gpu(gpu, cu, monkeypatch):
  """As test_starts_that_fall_gpu, over bf16 pages."""
  monkeypatch.setattr(K, "mx_prompt_direct", lambda *a: False)
  s = Seqs("mxfp8", [70, 33, 130], 2, 128, dev=gpu)
  q = torch.randn(40, 4, 128, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(gpu)
  whole = torch.full((80, 4, 128), 7.0, dtype=torch.bfloat16, device=gpu)
  for most in (40, 400):
    K.attn_prefill_mx(q, s.k, s.v, s.tables, torch.tensor(cu, dtype=torch.int32, device=gpu), s.ctx, most, 0.125, out=whole[20:60])
    assert (whole[:20] == 7).all() and (whole[60:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,Dh", [("mxfp4", 128), ("mxfp8", 128), ("mxfp4", 64), ("mxfp8", 64)])
def test_long_contexts_gpu(gpu, fmt, Dh):
  """Contexts past 128 pages as the rule itself cuts them, beside short ones; a workspace made for shorter ones; a few new tokens behind them."""
  s = Seqs(fmt, [32000, 33, 0, 8256], 1, Dh, dev=gpu)
  assert K.MXDecodeWorkspace.parts(4, 1, 500)[1] > 4
  for max_ctx in (32000, 4096, 64):
    check_decode(s, 4, Dh ** -0.5, ws=K.MXDecodeWorkspace(4, 4, 1, Dh, max_ctx, gpu))
  check_decode(s, 4, Dh ** -0.5)
  check_prompt(s, [3, 5, 0, 9], 4, Dh ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_long_context_among_many_gpu(gpu, fmt):
  """Pairs enough to fill the chip uncut: a context past 128 pages is cut all the same, the others stay whole."""
  lens = [5 + 7 * (b % 9) for b in range(64)]
  lens[40] = 9000
  s = Seqs(fmt, lens, 8, 64, dev=gpu)
  assert K.MXDecodeWorkspace.parts(64, 8, 141) == (71, 2)
  check_decode(s, 16, 0.125)
  check_decode(s, 16, 0.125, ws=K.MXDecodeWorkspace(64, 16, 8, 64, 4096, gpu))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,Dh", [("mxfp4", 128), ("mxfp8", 128), ("mxfp4", 64), ("mxfp8", 64)])
def test_far_rows_among_others_gpu(gpu, fmt, Dh, monkeypatch):
  """Far rows in some waves of a unit only, results where their queries were: the same as far rows and others by themselves."""
  H, Hkv = 4, 2
  s = Seqs(fmt, [300, 90], Hkv, Dh, dev=gpu)
  q = torch.randn(390, H, Dh, generator=torch.Generator().manual_seed(5))
  q[17], q[40:60], q[389, 1] = q[17] * 2.0 ** 90, q[40:60] * 2.0 ** 40, q[389, 1] * 2.0 ** 30
  q = q.to(torch.bfloat16)
  cu = torch.tensor([0, 300, 390], dtype=torch.int32, device=gpu)
  for tiles in (True, False):
    monkeypatch.setattr(K, "mx_prompt_tiles", lambda *a: tiles)
    whole = K.attn_prefill_mx(q.to(gpu), s.k, s.v, s.tables, cu, s.ctx, 300, 0.1)
    own = q.to(gpu)
    assert torch.equal(K.attn_prefill_mx(own, s.k, s.v, s.tables, cu, s.ctx, 300, 0.1, out=own), whole)
    assert torch.isfinite(whole).all()
    for rows, b, past in ((slice(0, 17), 0, 0), (slice(18, 40), 0, 18), (slice(60, 300), 0, 60), (slice(300, 389), 1, 0)):
      n = rows.stop - rows.start
      kv = [t[:past + n] for t in s.kv[b]]
      close(whole[rows], *attend64(q[rows], *kv, 0.1, past))
    for t, h in ((17, 0), (45, 3), (389, 1)):  # a far row takes its largest score's value: scores apart by far more than their error
      b, past = (0, t) if t < 300 else (1, t - 300)
      k, v = (x[:past + 1, h // (H // Hkv)] for x in s.kv[b])
      score = k @ q[t, h].double()
      first, second = score.topk(2).values
      if first - second > 2.0 ** -12 * (k.abs() @ q[t, h].double().abs()).max():
        assert torch.allclose(whole[t, h].double().cpu(), v[score.argmax()], rtol=2.0 ** -8, atol=0)
