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
  """The kernels and graphs on the pools in 8 or 4 bits against the bf16 kernels, eager, on pools with the same values."""
  got = play(runner(name, gpu, fmt), name)
  held_in_bf16(monkeypatch, fmt)
  want = play(runner(name, gpu, "bf16", use_graphs=False), name)
  for a, b in zip(got, want):
    assert torch.allclose(a, b, atol=2e-2, rtol=2e-2)


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
