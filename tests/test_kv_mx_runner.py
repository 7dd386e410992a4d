"""ShardRunner on a KV cache in 8 or 4 bits: against the same model on a bf16 cache that holds the same values, prompts in portions, mixed
steps, decode graphs, split shards, sizes, and the models it refuses."""
import pytest
import torch

from xotorch_support_jetson_amd.inference.shard import Shard
from xotorch_support_jetson_amd.main import build_parser
from xotorch_support_jetson_amd.models import transformer
from xotorch_support_jetson_amd.models.config import preset
from xotorch_support_jetson_amd.models.transformer import KVCache
from xotorch_support_jetson_amd.ops import kernels as K
from xotorch_support_jetson_amd.ops import reference as ref
from xotorch_support_jetson_amd.ops.linear import linear
from xotorch_support_jetson_amd.runtime.runner import ShardRunner

FMTS = ("mxfp8", "mxfp4")


def runner(name, dev, kv_dtype, lo=0, hi=None, **kw):
  c = preset(name)
  hi = c.num_layers - 1 if hi is None else hi
  return ShardRunner(c, Shard(name, lo, hi, c.num_layers), dev, **({"max_batch": 8, "max_ctx": 512, "seed": 3} | kw), kv_dtype=kv_dtype)


def tokens(name, n, seed=5):
  return torch.randint(0, preset(name).vocab_size, (n,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


def held_in_bf16(monkeypatch, fmt):
  """linear_rope_kv for bf16 pools that writes the values a pool of this format would hold."""
  def write(x, w, bias, pos, cos_sin, slots, kc, vc, H, Hkv, wide=True):
    qkv = linear(x, w, bias=bias)
    n, Dh = kc.shape[0], kc.shape[-1]
    k, v = (torch.zeros(n, Hkv, K.mx_page_bytes(fmt, Dh), dtype=torch.uint8, device=kc.device) for _ in range(2))
    q = K.rope_kv_write_mx(qkv, pos, cos_sin, slots, k, v, H, Hkv)
    ok = slots >= 0
    s = slots[ok].long()
    kv = [t[s // 64, :, s % 64] for t in ref.mx_read(k, v, torch.arange(n, device=kc.device), Dh)]
    ref.write_kv(*kv, s, kc, vc)
    return q
  monkeypatch.setattr(transformer, "linear_rope_kv", write)


def play(r, name):
  """A prompt, another with the first one's next token (a mixed step), a portion behind a cached prefix, decode steps."""
  ids = tokens(name, 400)
  outs = []

  def step(rids, lens, at):  # (a graph's logits are its own buffer: copied before the next step)
    outs.append(r.forward(rids, lens, ids[at:at + sum(lens)]).float().cpu().clone())
  step(["a"], [70], 0)
  step(["a", "b"], [1, 130], 70)
  step(["b"], [20], 201)
  for i in range(4):
    step(["a", "b"], [1, 1], 230 + 2 * i)
  step(["b"], [1], 300)
  return outs


@pytest.mark.parametrize("fmt", FMTS)
def test_same_values_cpu(fmt, monkeypatch):
  got = play(runner("tiny-llama-d64", "cpu", fmt), "tiny-llama-d64")
  held_in_bf16(monkeypatch, fmt)
  want = play(runner("tiny-llama-d64", "cpu", "bf16"), "tiny-llama-d64")
  for a, b in zip(got, want):
    assert torch.allclose(a, b, atol=2e-2, rtol=2e-2)


@pytest.mark.parametrize("fmt", FMTS)
def test_close_to_bf16_cpu(fmt):
  for a, b in zip(play(runner("tiny-phi3", "cpu", fmt), "tiny-phi3"), play(runner("tiny-phi3", "cpu", "bf16"), "tiny-phi3")):
    assert torch.corrcoef(torch.stack([a.flatten(), b.flatten()]))[0, 1] > 0.95


def test_sizes_and_choice(monkeypatch):
  c = preset("tiny-llama")
  whole = KVCache.bytes_per_page(c, 4)
  assert KVCache.bytes_per_page(c, 4, kv_dtype="mxfp8") * 64 == whole * 33 and KVCache.bytes_per_page(c, 4, kv_dtype="mxfp4") * 64 == whole * 17
  monkeypatch.setenv("XOT_KV_DTYPE", "mxfp4")
  r = runner("tiny-llama", "cpu", None)
  assert r.kv_dtype == "mxfp4" and r.kv.k.dtype == torch.uint8
  assert r.kv.nbytes() == KVCache.bytes_per_page(c, 4, kv_dtype="mxfp4") * r.kv.num_pages
  assert runner("tiny-llama", "cpu", "bf16").kv.k.dtype == torch.bfloat16
  assert build_parser().parse_args(["run", "tiny-llama", "--kv-dtype", "mxfp8"]).kv_dtype == "mxfp8"


@pytest.mark.parametrize("name,fmt", [("tiny-deepseek-v2", "mxfp8"), ("tiny-tarepel", "mxfp4"), ("tiny-llama", "int4")])
def test_refused(name, fmt):
  with pytest.raises(ValueError, match="kv_dtype"):
    runner(name, "cpu", fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("name", ["tiny-llama-d64", "tiny-phi3", "tiny-qwen"])
def test_same_values_gpu(gpu, name, fmt, monkeypatch):
  """Every attention of a model's steps against the bf16 kernels on the same queries and the pages read back.  (Call by call: two whole
  runs drift apart by more than either kernel's error.  Where the first layers' sums differ by d = 2^-8 of a value, a value that stands near
  the border between two elements, d of every step of them, moves by a whole step; a step is a quarter of the value in mxfp4, so its keys and
  values differ by sqrt(2^-8 / 4) = 2^-5 of themselves in the mean square, eight times what the sums did.)  Each side rounds its weights and
  its result to bf16, 2^-8 each of sum p |v| and of the result; the scores' errors are below 2^-9 of the former (tests/test_kv_mx.py)."""
  attention = transformer.ShardModel._attention
  calls = []

  def checked(self, q, li, inp, ws=None, **kw):
    out = attention(self, q, li, inp, ws, **kw)
    kc, vc, W = self.kv.k[li], self.kv.v[li], inp.block_tables.shape[1]
    k, v = K.kv_read_mx(kc, vc, inp.block_tables, inp.ctx_lens, q.shape[-1])
    own = torch.arange(k.shape[0], dtype=torch.int32, device=q.device).view(-1, W)
    want, weight = (K.attn_decode(q, k, t, own, inp.ctx_lens, self.scale) if inp.decode else
                    K.attn_prefill(q, k, t, own, inp.cu_q, inp.ctx_lens, inp.max_qlen, self.scale) for t in (v, v.abs()))
    tol = 2.0 ** -7 * want.float().abs() + (2.0 ** -7 + 2.0 ** -8) * weight.float() + 1e-30
    calls.append(((out.view(want.shape).float() - want.float()).abs() / tol).max().item())
    return out
  monkeypatch.setattr(transformer.ShardModel, "_attention", checked)
  outs = play(runner(name, gpu, fmt, use_graphs=False), name)
  assert all(torch.isfinite(t).all() for t in outs)
  assert len(calls) == 8 * preset(name).num_layers and max(calls) <= 1.0, max(calls)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_graphs_and_shards_gpu(gpu, fmt):
  """Replayed steps against eager ones, twice over, with other batches between; two shards against one."""
  name = "tiny-llama"
  g, e = runner(name, gpu, fmt), runner(name, gpu, fmt, use_graphs=False)
  first, second = runner(name, gpu, fmt, 0, 1), runner(name, gpu, fmt, 2, 3)
  ids, lens = tokens(name, 300), [3, 64, 130]
  rids = ["a", "b", "c"]
  n = sum(lens)
  for r in (g, e):
    r.forward(rids, lens, ids[:n])
  second.forward(rids, lens, first.forward(rids, lens, ids[:n]))
  for step in range(6):
    some = rids[: 1 + step % 3]
    x = ids[200 + step:200 + step + len(some)]
    ones = [1] * len(some)
    a, b = g.forward(some, ones, x).clone(), e.forward(some, ones, x)
    c = second.forward(some, ones, first.forward(some, ones, x))
    torch.cuda.synchronize()
    assert torch.allclose(a, b, atol=2e-2, rtol=2e-2) and torch.allclose(a, c, atol=2e-2, rtol=2e-2)


@pytest.mark.gpu
def test_routed_model_gpu(gpu):
  got, want = (play(runner("tiny-mixtral", gpu, d), "tiny-mixtral") for d in ("mxfp8", "bf16"))
  for a, b in zip(got, want):
    assert torch.corrcoef(torch.stack([a.flatten(), b.flatten()]))[0, 1] > 0.9


@pytest.mark.parametrize("fmt", ("mxfp8", "bf16"))
def test_steps_know_their_longest_context(fmt, monkeypatch):
  seen = []
  attention = transformer.ShardModel._attention

  def looked(self, q, li, inp, *a, **kw):
    seen.append((inp.max_ctx, int(inp.ctx_lens.max()), inp.block_tables.shape[1]))
    return attention(self, q, li, inp, *a, **kw)
  monkeypatch.setattr(transformer.ShardModel, "_attention", looked)
  play(runner("tiny-llama-d64", "cpu", fmt, max_ctx=4096), "tiny-llama-d64")
  assert len(seen) == 8 * preset("tiny-llama-d64").num_layers and all(a == b < 200 and w == 64 for a, b, w in seen)


def test_table_widths_of_graphs():
  """Classes of block tables that decode graphs are captured with: on to the longest context where no plan cuts contexts by their lengths."""
  assert runner("tiny-llama", "cpu", "mxfp8", max_ctx=9000, num_pages=64)._widths == [8, 16, 32, 64, 128, 141]
  assert runner("tiny-llama", "cpu", "mxfp4", max_ctx=512, num_pages=64)._widths == [8]
  assert runner("tiny-llama", "cpu", "bf16", max_ctx=9000, num_pages=64)._widths == [8, 16, 32, 141]
  assert runner("tiny-llama", "cpu", "bf16", max_ctx=1024, num_pages=64)._widths == [8, 16]


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["tiny-mixtral", "tiny-llama"])
def test_routed_projections_keep_their_order_gpu(gpu, name, monkeypatch):
  """From 17 rows on a routed model's query, key and value projection never takes the GEMM whose sums run in another order, as
  linear_rope_kv(wide=False) (a token whose experts are almost tied turns on the last bits); other models' may."""
  from xotorch_support_jetson_amd.ops import linear as linear_mod
  choose, asked = linear_mod.policy.shuffled_cfg, []
  r = runner(name, gpu, "mxfp8", use_graphs=False)

  def looked(x, w, *a, **kw):
    if any(w is t.qkv_w for t in r.weights.layers.values()):
      asked.append((x.shape[0], kw.get("wave", "")))
    return choose(x, w, *a, **kw)
  monkeypatch.setattr(linear_mod.policy, "shuffled_cfg", looked)
  r.forward(["a", "b"], [4, 5], tokens(name, 9))
  r.forward(["c"], [40], tokens(name, 40))
  assert set(asked) == {(9, "y"), (40, "" if preset(name).num_experts else "y")}


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_graphs_of_wider_tables_gpu(gpu, fmt):
  """Replayed steps across the classes past 32 pages against eager ones whose forms are chosen for the same class (so that sums run in the same
  order: what quantising makes of another order's rounding is in test_same_values_gpu)."""
  name = "tiny-llama"
  g, e = (runner(name, gpu, fmt, max_ctx=9000, max_batch=2, num_pages=200, use_graphs=u) for u in (None, False))
  prepare = e._prepare

  def by_class(*a):
    inp = prepare(*a)
    if inp.decode:
      inp.max_ctx = 64 * next(w for w in g._widths if 64 * w >= inp.max_ctx)
    return inp
  e._prepare = by_class
  ids = tokens(name, 4090)
  for r in (g, e):
    r.forward(["a"], [2045], ids[:2045])
    r.forward(["b"], [70], ids[:70])

  def step(x):
    a, b = g.forward(["a", "b"], [1, 1], x).clone(), e.forward(["a", "b"], [1, 1], x)
    assert torch.isfinite(a).all() and torch.allclose(a, b, atol=2e-2, rtol=2e-2)
  for i in range(6):  # 2046 to 2051 tokens: 32 pages, then 33
    step(ids[i:i + 2])
  assert [w for _, w in g._graphs] == [32, 64]
  for r in (g, e):
    r.forward(["a"], [2050], ids[2000:4050])
  step(ids[9:11])
  assert [w for _, w in g._graphs] == [32, 64, 128]
