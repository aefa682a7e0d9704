"""Streamed global attention: frames arrive one after another.

* ``BlockCache`` holds the keys and values of what was seen, in 8 bits or 4,
  in pages of 64 tokens that a page table hands to the sequences;
  ``PagePool`` counts who holds which page, so that sequences can share them.
* ``stream_attention`` is a global layer over the new frames' tokens: their
  keys and values are written into the cache, patch queries attend to the
  pages that a cheap score chooses for each block of 128 of them, special
  tokens to everything seen (as in ``adaptive_sparse_attention_forward``,
  which needs the whole clip at once).
* ``AggregatorStream`` runs a VGGT-shaped ``Aggregator`` that way: ``push``
  takes the next frames, whose global blocks see all frames so far; ``fork``
  branches off, ``keep`` forgets frames.
"""
from __future__ import annotations

import math

import torch

from . import ops
from .pipeline import ratio_to_topk


class BlockCache:
    """Keys and values of ``heads`` key heads in 8 bits or 4, ``pages`` pages of 64 tokens.

    ``kc`` / ``vc``: the codes, e4m3 or e2m1 (values transposed within a
    page), ``ks`` / ``vs``: the rows' powers of two, with 4 bits one for each 32
    features of a key row, and ``vo`` for those of a value row; ``mean``: each
    page's mean key in bf16 (``include/vasc_stream.h`` has the layout).
    ``ops.cache_write`` fills it, ``ops.cache_read`` / ``cache_select`` /
    ``cache_attn`` read it, ``cache_copy`` / ``cache_compact`` move what it holds.
    Which pages belong to whom is the caller's page table, which a ``PagePool``
    can keep. The cache starts as zeros.
    """

    def __init__(self, pages: int, heads: int, head_dim: int, device="cuda", bits: int = 8):
        if pages < 1 or heads < 1:
            raise ValueError(f"a cache needs pages and heads, got {pages} and {heads}")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim {head_dim} not built (64, 128)")
        if bits not in (4, 8):
            raise ValueError(f"bits {bits} not built (4, 8)")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("the block cache lives on a GPU (the HIP path has no CPU fallback)")
        self.pages, self.heads, self.head_dim, self._bits = int(pages), int(heads), int(head_dim), int(bits)
        u8 = dict(device=device, dtype=torch.uint8)
        page = ops.BLOCK_K
        if bits == 8:
            self._kc = torch.zeros(pages, heads, page, head_dim, **u8)
            self._vc = torch.zeros(pages, heads, head_dim, page, **u8)
            self._ks = torch.zeros(pages, heads, page, **u8)
            self._vo = None
        else:
            self._kc = torch.zeros(pages, heads, page * head_dim // 2, **u8)
            self._vc = torch.zeros(pages, heads, page * head_dim // 2, **u8)
            self._ks = torch.zeros(pages, heads, head_dim // 32, page, **u8)
            self._vo = torch.zeros(pages, heads, head_dim, **u8)
        self._vs = torch.zeros(pages, heads, page, **u8)
        self._mean = torch.zeros(pages, heads, head_dim, device=device, dtype=torch.bfloat16)
        self._locate()

    def _locate(self) -> None:
        """The buffers stay where they are, so a call need not ask for their addresses again."""
        if not self._kc.is_cuda:
            raise ValueError("the block cache lives on a GPU (the HIP path has no CPU fallback)")
        self.device_index = self._kc.get_device()
        self.pointers = tuple(t.data_ptr() for t in (self._kc, self._vc, self._ks, self._vs, self._vo) if t is not None)
        self.mean_pointer = self._mean.data_ptr()

    def __setstate__(self, state: dict) -> None:
        """A copy or an unpickled cache: the state's addresses are the original's."""
        self.__dict__.update({"_bits": 8, "_vo": None, **state})
        self._locate()

    bits = property(lambda self: self._bits)
    kc = property(lambda self: self._kc)
    vc = property(lambda self: self._vc)
    ks = property(lambda self: self._ks)
    vs = property(lambda self: self._vs)
    vo = property(lambda self: self._vo)
    mean = property(lambda self: self._mean)

    @property
    def nbytes(self) -> int:
        """Bytes of device memory: a value pair has 2 + 2/D bytes, with 4 bits 1 + 3/64 + 1/D, and a page its means."""
        return sum(t.numel() * t.element_size() for t in (self.kc, self.vc, self.ks, self.vs, self.vo, self.mean)
                   if t is not None)


class PagePool:
    """Who holds the pages of one or more block caches that a page table serves.

    ``refs [pages]`` int32 on the GPU counts each page's holders, the entries
    of page tables that name it: a page is free where it is not positive, also
    where an entry names it that no operator has put there.
    ``ops.pages_reserve`` gives sequences the lowest free pages, ``pages_fork``
    lets sequences share pages, ``pages_free`` gives them back; a table starts
    as -1 throughout. Nothing is kept on the host, so that a captured call
    serves every step. Calls on one pool go one after another: on one stream,
    or on streams that wait for each other.
    """

    def __init__(self, pages: int, device="cuda"):
        if not 1 <= pages < 1 << 26:
            raise ValueError(f"a pool has 1 to 2^26 - 1 pages, got {pages}")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("the page pool lives on a GPU (the HIP path has no CPU fallback)")
        self.pages = int(pages)
        self._refs = torch.zeros(pages, device=device, dtype=torch.int32)
        self._locate()

    def _locate(self) -> None:
        if not self._refs.is_cuda:
            raise ValueError("the page pool lives on a GPU (the HIP path has no CPU fallback)")
        self.device_index, self.pointer = self._refs.get_device(), self._refs.data_ptr()

    def __setstate__(self, state: dict) -> None:
        """A copy or an unpickled pool: the state's address is the original's."""
        self.__dict__.update(state)
        self._locate()

    refs = property(lambda self: self._refs)

    def available(self) -> int:
        """Free pages; waits for the GPU."""
        return int((self._refs <= 0).sum())


def _layer_qkv(attn, x: torch.Tensor, pos: torch.Tensor | None, frames: int, special: int) -> tuple:
    """q of the patch and of the special tokens, k and v ``[B,H,*,D]`` in bf16, normed and turned."""
    from .aggregator import RotaryPositionEmbeddingAxes, fused_layout_supported, head_norm, layer_norm_args
    B, T, dim = x.shape
    H = attn.num_heads
    D = dim // H
    qkv = attn.qkv(x).to(torch.bfloat16).view(B, T, 3, H, D)
    q, k, v = qkv.unbind(2)
    rope = getattr(attn, "rope", None)
    if fused_layout_supported(attn):
        turned = rope is not None and pos is not None
        return ops.pack_qkv(q, k, v, frames, T // frames, special, q_norm=layer_norm_args(attn.q_norm),
                            k_norm=layer_norm_args(attn.k_norm), pos=pos if turned else None,
                            rope_tables=rope.tables(D, x.device) if turned else None)
    q, k = head_norm(attn.q_norm, q.transpose(1, 2)), head_norm(attn.k_norm, k.transpose(1, 2))
    if rope is not None and pos is not None:
        if isinstance(rope, RotaryPositionEmbeddingAxes):
            q, k = rope.rotate(q, k.to(q.dtype), pos)
        else:
            q, k = rope(q, pos), rope(k, pos)
    return ops.pack_qkv(*(t.to(torch.bfloat16).transpose(1, 2) for t in (q, k)), v, frames, T // frames, special)


@torch.no_grad()
def stream_attention(attn, x: torch.Tensor, pos: torch.Tensor | None, cache: BlockCache, page_table: torch.Tensor,
                     start: torch.Tensor, lengths: torch.Tensor, *, keep: int | None, frames: int = 1, special: int = 0,
                     block_q: int = ops.BLOCK_Q, sink: int = 1, recent: int = 1) -> torch.Tensor:
    """Global attention of new tokens over everything in the cache, them included.

    ``attn``: an ``aggregator.Attention`` (or a module with its fields); x
    ``[B,T,dim]``: ``frames`` frames of ``T / frames`` tokens, the first
    ``special`` of each of them special; pos ``[B,T,2]`` (or as many axes as
    the module's rope has). ``start [B]``: tokens of each sequence in the
    cache before the call, ``lengths [B]``: after it (``start + T``); both stay
    on the device, so that a captured call serves every step. ``keep``: pages
    that a block of patch queries chooses beside the first ``sink`` and the
    last ``recent``; None: all. A call's tokens are held in the global layers'
    order, all patches before all special tokens. Returns ``[B,T,dim]``. No
    gradients.
    """
    ops._inference(x, "x")
    dev = ops._gpu(x, "x")
    if pos is not None:
        ops._gpu(pos, "pos", dev)
    B, T, dim = x.shape
    if frames < 1 or T < 1 or T % frames or not 0 <= special <= T // frames:
        raise ValueError(f"{T} tokens are not {frames} frames with {special} special tokens each")
    H = attn.num_heads
    with ops.on_device(dev):
        q_patch, q_special, k, v = _layer_qkv(attn, x, pos, frames, special)
        ops.cache_write(cache, k, v, page_table, start)
        if keep is None:
            o_patch = ops.cache_attn(q_patch, cache, page_table, lengths)
        else:
            index, count = ops.cache_select(q_patch, cache, page_table, lengths, keep, block_q=block_q, sink=sink,
                                            recent=recent)
            o_patch = ops.cache_attn(q_patch, cache, page_table, lengths, index, count, block_q=block_q)
        o_special = ops.cache_attn(q_special, cache, page_table, lengths) if q_special is not None else None
        if o_patch.shape[2]:
            out = ops.restore_tokens(o_patch, o_special, frames, T // frames, special)
        else:  # frames of special tokens only, which are in order
            out = o_special.transpose(1, 2).reshape(B, T, H * (dim // H))
        out = attn.proj(out.to(x.dtype))
        drop = getattr(attn, "proj_drop", None)
        return drop(out) if drop is not None else out


class AggregatorStream:
    """Frames one after another through a VGGT-shaped ``aggregator.Aggregator``.

    ``push(images)`` takes the next frames ``[B,n,3,H,W]`` (the same B, H and W
    every time) and returns what the aggregator returns for them. Frame blocks
    see their frame, global blocks all frames held, through a cache a layer
    (``bits`` 8 or 4); a block of 128 patch queries keeps ``1 - sparse_ratio`` of
    the pages. The model's own global attention (``Attention`` or an installed
    sparse one) is not used. ``reset()`` starts over.

    ``fork()`` gives another stream that goes on from here, with the frames so
    far in pages that both share; up to ``branches`` streams at once, each of
    at most ``max_frames`` frames (the caches hold so many), until
    ``close()``. ``keep(frames)`` forgets the frames that it does not list; it
    needs free pages for those that stay, so a stream that forgets when it
    holds n frames and keeps m of them wants ``max_frames`` n + m + 1 (frames of
    64 tokens or more). Streams that share caches are called one after another,
    as the pool's operators; the pool is theirs alone.
    """

    def __init__(self, model, max_frames: int, *, sparse_ratio: float = 0.75, sink: int = 1, recent: int = 1, bits: int = 8,
                 branches: int = 1):
        if max_frames < 1 or not 0.0 <= sparse_ratio < 1.0:
            raise ValueError(f"max_frames {max_frames} must be positive, sparse_ratio {sparse_ratio} in [0, 1)")
        if bits not in (4, 8) or branches < 1:
            raise ValueError(f"bits {bits} must be 4 or 8, branches {branches} positive")
        self.model, self.max_frames, self.sparse_ratio = model, int(max_frames), float(sparse_ratio)
        self.sink, self.recent, self.bits, self.branches = sink, recent, int(bits), int(branches)
        self.caches: list[BlockCache] = []
        self.pool: PagePool | None = None
        self.frames, self._shape = 0, None
        self._seen = 0      # frames pushed, those that were forgotten among them: the next one's time
        self._tokens = []   # of each frame held, the (first, number) of its runs of tokens
        self._streams = [1]  # open streams of these caches, shared among them
        self._forked = False  # whether another stream may hold this one's last page

    def _open(self) -> None:
        if self._streams is None:
            raise ValueError("the stream is closed")

    def reset(self) -> None:
        self._open()
        if self.pool is not None:  # whatever is held: a push that failed has reserved pages, too
            with ops.on_device(self.pool.device_index):
                ops.pages_free(self.pool, self.page_table, self.lengths)
        self.frames = self._seen = 0
        self._tokens, self._forked = [], False

    def close(self) -> None:
        """Gives the stream's pages back; of no use after it."""
        if self._streams is not None:
            self.reset()
            self._streams[0] -= 1
            self._streams = None

    def fork(self) -> "AggregatorStream":
        """Another stream with the frames so far; pages are copied where one of the two goes on in them."""
        self._open()
        if not self.frames:
            raise ValueError("nothing to fork: no frame has been pushed")
        if self._streams[0] >= self.branches:
            raise ValueError(f"the stream was made for {self.branches} branches")
        other = AggregatorStream.__new__(AggregatorStream)
        other.__dict__.update(self.__dict__, _tokens=list(self._tokens))
        with ops.on_device(self.pool.device_index):
            source = torch.arange(self.page_table.shape[0], device=self.page_table.device, dtype=torch.int32)
            other.page_table, other.lengths = ops.pages_fork(self.pool, self.page_table, self.lengths, source)
        self._streams[0] += 1
        self._forked = other._forked = True
        return other

    def keep(self, frames) -> None:
        """Forgets all frames but the listed ones (places among those held, ascending); their tokens move to free pages, of
        which there must be enough for them beside all that are held. Waits for the GPU."""
        self._open()
        frames = [int(f) for f in frames]
        if not frames or any(b <= a for a, b in zip(frames, frames[1:])) or frames[0] < 0 or frames[-1] >= self.frames:
            raise ValueError(f"frames {frames} must be some of the {self.frames} held, ascending")
        if len(frames) == self.frames:
            return
        B, mp = self.page_table.shape
        P = self._shape[1]
        n = len(frames) * P
        with torch.no_grad(), ops.on_device(self.pool.device_index):
            need = B * math.ceil(n / ops.BLOCK_K)
            free = self.pool.available()
            if need > free:
                raise ValueError(f"{len(frames)} frames need {need} free pages to move to, {free} are: allow more frames")
            runs = [run for f in frames for run in self._tokens[f]]
            index = torch.cat([torch.arange(at, at + m, dtype=torch.int32) for at, m in runs]).to(self.page_table.device)
            table, lengths = torch.full_like(self.page_table, -1), torch.zeros_like(self.lengths)
            granted, _, _ = ops.pages_reserve(self.pool, table, lengths, n)
            try:
                for cache in self.caches:
                    ops.cache_compact(cache, self.page_table, index.expand(B, n), table)
            except BaseException:  # the frames are still where they were
                ops.pages_free(self.pool, table, lengths)
                raise
            ops.pages_free(self.pool, self.page_table, self.lengths)
            self.page_table, self.lengths = table, granted.clone()
        at, tokens = 0, []
        for f in frames:
            tokens.append([])
            for _, m in self._tokens[f]:
                tokens[-1].append((at, m))
                at += m
        self.frames, self._tokens, self._forked = len(frames), tokens, False

    def _begin(self, B: int, P: int, hw: tuple, device) -> None:
        if self._shape is None or self._shape[:3] != (B, P, hw) or self._shape[3] != device:
            if self.frames or self._streams[0] > 1:
                raise ValueError(f"frames of another batch, size or device: {(B, P, hw, device)} after {self._shape}")
            pages = math.ceil(self.max_frames * P / ops.BLOCK_K)
            attn = self.model.global_blocks[0].attn
            total = B * pages * self.branches
            self.caches = [BlockCache(total, attn.num_heads, attn.head_dim, device, self.bits) for _ in self.model.global_blocks]
            self.pool = PagePool(total, device)
            self.page_table = torch.full((B, pages), -1, device=device, dtype=torch.int32)
            self.lengths = torch.zeros(B, device=device, dtype=torch.int32)
            self._shape = (B, P, hw, device)

    @torch.no_grad()
    def push(self, images: torch.Tensor):
        """images ``[B,n,3,H,W]`` in [0, 1] -> (list of per-layer outputs, patch_start_idx)."""
        self._open()
        with ops.on_device(ops._gpu(images, "images")):
            return self._push(images)

    def _push(self, images: torch.Tensor):
        from .aggregator import grid_positions, patch_tokens, RotaryPositionEmbeddingAxes
        m = self.model
        B, n, _, Hi, Wi = images.shape
        if n < 1 or self.frames + n > self.max_frames:
            raise ValueError(f"{n} more frames after {self.frames}: the stream holds {self.max_frames}")
        x = ((images - m._resnet_mean) / m._resnet_std).reshape(B * n, 3, Hi, Wi).to(m.patch_embed.weight.dtype)
        tokens = patch_tokens(m.patch_embed, x)

        def expand(token):  # the stream's first frame has tokens of its own
            if self._seen == 0:
                return m._expand(token, B, n)
            return token[:, 1:].expand(B, n, *token.shape[2:]).reshape(B * n, *token.shape[2:])

        special = [expand(m.register_token)]
        if m.camera_token is not None:
            special.insert(0, expand(m.camera_token))
        tokens = torch.cat([*(s.to(tokens.dtype) for s in special), tokens], dim=1)
        h, w = Hi // m.patch_size, Wi // m.patch_size
        P, C, S = tokens.shape[1], tokens.shape[2], m.patch_start_idx
        self._begin(B, P, (h, w), tokens.device)
        pos = grid_positions(B * n, h, w, S, images.device).to(torch.int32).contiguous()
        if isinstance(m.global_blocks[0].attn.rope, RotaryPositionEmbeddingAxes):
            # (frame, row, column)
            t = torch.arange(self._seen, self._seen + n, device=images.device, dtype=torch.int32)
            pos = torch.cat([t.repeat(B).view(B * n, 1, 1).expand(-1, P, -1), pos], -1).contiguous()
        pos_global = pos.view(B, n * P, -1)
        before, after = self.frames * P, (self.frames + n) * P
        start = self.lengths
        # there are pages for `branches` streams of max_frames frames, and no stream holds more, a failed push's among
        # them: everything is granted
        granted, src, dst = ops.pages_reserve(self.pool, self.page_table, start, n * P)
        if self._forked:
            for cache in self.caches:
                ops.cache_copy(cache, src, dst)
        lengths = start + granted
        pages = math.ceil(after / ops.BLOCK_K)
        keep = None if self.sparse_ratio == 0 else max(0, ratio_to_topk(pages, self.sparse_ratio) - self.sink - self.recent)
        outputs, normed = [], None
        for i in range(m.aa_block_num):
            fb, gb = m.frame_blocks[i], m.global_blocks[i]
            tokens, normed = fb(tokens.view(B * n, P, C), pos=pos, normed=normed, next_norm=gb.norm1)
            frame_out = tokens.view(B, n, P, C)

            def attend(attn, y, at, cache=self.caches[i]):
                return stream_attention(attn, y, at, cache, self.page_table, start, lengths, keep=keep, frames=n,
                                        special=S, sink=self.sink, recent=self.recent)

            nxt = m.frame_blocks[i + 1].norm1 if i + 1 < m.aa_block_num else None
            out = gb(tokens.view(B, n * P, C), pos=pos_global, normed=normed.view(B, n * P, C), next_norm=nxt, attend=attend)
            tokens, normed = out if nxt is not None else (out, None)
            if normed is not None:
                normed = normed.view(B * n, P, C)
            outputs.append(torch.cat([frame_out, tokens.view(B, n, P, C)], dim=-1) if i in m.intermediate_layer_idx else None)
        # a call's tokens are held all patches before all special tokens
        self._tokens += [[(before + j * (P - S), P - S), (before + n * (P - S) + j * S, S)] for j in range(n)]
        self.lengths, self._forked = lengths, False
        self.frames += n
        self._seen += n
        return outputs, S
