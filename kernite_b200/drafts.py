"""A decode stack that checks drafted tokens: its weights read once for up to 8 tokens of a tree.

A step of :class:`DraftStack` takes T drafted tokens of one sequence. Draft i continues draft
parents[i] (-1: the kept context), so that several continuations are checked at once; T = 1 is a plain
decode step, and a prompt is a chain of drafts that are all kept. Per layer of the stack's configuration:

    q|k|v      one matvec for T vectors
    write      q rotated, k rotated and kept, v kept: draft i in the cache's row after the context + i,
               turned by its own position (the context's length + its depth in the tree)
    attention  every draft over the context and over the drafts above it
    o, gate|up, down  one matvec each for T vectors

then the head. :func:`accepted` walks the tree along the model's own choices, and :meth:`DraftStack.keep`
moves the rows of the drafts that were right to the end of the context.

kernite has no decode stack; the layers are those of kernite_b200.stack, with the paged 16-, 8- or
4-bit cache in the place of its f16 one.
"""
from __future__ import annotations

import contextlib
import math

from .stack import CudaBackend, StackConfig, plan

MAX_DRAFTS = 8  # what one matvec of a Q6_K matrix takes


def tree_words(parents) -> tuple[list[int], list[int]]:
    """(mask words, depths) of a tree: bit u of word t says that draft t sees draft u, which it does for
    itself and for those above it."""
    words, depths = [], []
    for i, up in enumerate(parents):
        if not -1 <= up < i:
            raise ValueError(f"draft {i}'s parent {up} does not come before it")
        words.append((words[up] if up >= 0 else 0) | 1 << i)
        depths.append(depths[up] + 1 if up >= 0 else 0)
    return words, depths


def accepted(tokens, parents, root: int, choices) -> tuple[list[int], int]:
    """The drafts that greedy decoding keeps, in order, and the token after them. ``root`` is the token
    that the model chose after the context, ``choices[i]`` the one it chose after draft i."""
    path, want, at = [], root, -1
    for i, (token, up) in enumerate(zip(tokens, parents)):
        if up == at and token == want:
            path.append(i)
            want, at = int(choices[i]), i
    return path, want


class DraftStack:
    """One sequence's stack and caches on one GPU. ``cache``: CACHE_F16, CACHE_Q8 or CACHE_Q4;
    ``cfg.max_pos`` positions fit, drafts among them. The work of a call goes to ``stream`` (None: torch's
    current one at the call), after what the caller's current stream was given before the call, and what
    it is given afterwards waits for it."""

    def __init__(self, cfg: StackConfig, kernels, *, cache: int | None = None, page_size: int = 64,
                 max_drafts: int = MAX_DRAFTS, stream=None):
        import torch

        import kernite_b200 as kb

        if not 1 <= max_drafts <= MAX_DRAFTS:
            raise ValueError(f"max_drafts must be 1..{MAX_DRAFTS}")
        if cfg.hidden % cfg.head_dim or cfg.kv % cfg.head_dim or cfg.n_heads % cfg.n_kv:
            raise ValueError("attention needs whole heads and whole query groups")
        self.kb, self.torch, self.cfg, self.k, self.stream = kb, torch, cfg, kernels, stream
        self.max_drafts, self.page, self.kept, self.parents = max_drafts, page_size, 0, ()
        self.done = torch.cuda.Event()  # the last call's work
        self.shards = plan(cfg, 0, 1)
        load = lambda name, layer: backend.weights(self.shards[name], cfg.seed, cfg.tensor_id(layer, name))
        with self._ordered() as now:
            backend = CudaBackend(kernels, stream=now)
            self.weights = [{n: load(n, layer) for n in ("qkv", "o", "gate_up", "down")} for layer in range(cfg.layers)]
            self.head = load("head", cfg.layers)
            t, h = max_drafts, cfg.hidden
            vec = lambda n: torch.zeros(t, n, dtype=torch.float32, device="cuda")
            self.x, self.qkv, self.q, self.att, self.o = vec(h), vec(h + 2 * cfg.kv), vec(h), vec(h), vec(h)
            self.a, self.xd, self.logits = vec(cfg.ffn), vec(h), vec(cfg.vocab)
            kind = kb.CACHE_Q8 if cache is None else cache
            self.n_pages = -(-cfg.max_pos // page_size)
            nbytes = kb.cache_bytes(kind, cfg.n_kv, cfg.head_dim, page_size, self.n_pages)
            ints = lambda n, dtype: torch.zeros(n, dtype=dtype, device="cuda")
            self.pages = torch.arange(self.n_pages, dtype=torch.int32, device="cuda")
            self.positions, self.starts, self.prefix = (ints(n, torch.int32) for n in (t, 2, 1))
            self.slots, self.masks, self.src, self.dst = (ints(t, torch.int64) for _ in range(4))
            self.caches = [kb.KvCache(kind, cfg.n_kv, cfg.head_dim, page_size, self.n_pages,
                                      *(torch.zeros(nbytes, dtype=torch.uint8, device="cuda") for _ in "kv"))
                           for _ in range(cfg.layers)]
            self.rope = kb.Rope(cfg.head_dim, kb.ROPE_PAIRS, cfg.rope_base)
            need = kernels.tree_workspace(self._tree(self.caches[0], t, None, 0))
            self.workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
        self.descs = {}

    @contextlib.contextmanager
    def _ordered(self):
        """The stream that a call's work goes to, made torch's current one. It waits for the call before (whose
        stream may have been another) and for the caller's stream, which then waits for it."""
        cuda = self.torch.cuda
        caller = cuda.current_stream()
        stream = caller if self.stream is None else self.stream
        stream.wait_event(self.done)
        if stream != caller:
            stream.wait_stream(caller)
        try:
            with cuda.stream(stream):
                yield stream
        finally:
            self.done.record(stream)
            if stream != caller:
                caller.wait_event(self.done)

    def _tree(self, cache, drafts: int, workspace, nbytes: int):
        return self.kb.tree_desc(cache, self.att, self.q, self.cfg.n_heads, self.starts, self.prefix, self.pages,
                                 self.n_pages, 1, drafts, drafts, self.cfg.max_pos, mask=self.masks,
                                 workspace=workspace, workspace_bytes=nbytes)

    def _step_descs(self, drafts: int):
        """The layers' write and attention descriptors for this many drafts, made once."""
        if drafts not in self.descs:
            self.descs[drafts] = [
                (self.kb.cache_write_desc(c, self.rope, self.qkv, self.q, self.positions, self.slots, drafts,
                                          self.cfg.n_heads),
                 self._tree(c, drafts, self.workspace, self.workspace.numel())) for c in self.caches]
        return self.descs[drafts]

    def _put(self, to, values) -> None:
        to[: len(values)].copy_(self.torch.tensor(values, dtype=to.dtype))

    def check(self, x, parents):
        """Logits [T, vocab] after each of T drafts, whose input vectors are x [T, hidden] (f32, on the
        GPU). The drafts' rows are in the caches, and the logits in their buffer, until the next call; keep()
        makes the rows the context's."""
        cfg, kb, k, n = self.cfg, self.kb, self.k, len(parents)
        if not 1 <= n <= self.max_drafts:
            raise ValueError(f"1..{self.max_drafts} drafts a step")
        if tuple(x.shape) != (n, cfg.hidden):
            raise ValueError(f"x must be {n} vectors of {cfg.hidden}")
        if self.kept + n > cfg.max_pos:
            raise ValueError(f"the caches hold {cfg.max_pos} positions")
        words, depths = tree_words(parents)
        self.parents = ()  # nothing to keep until this step is whole
        with self._ordered() as stream:
            self.x[:n].copy_(x)
            self._put(self.positions, [self.kept + d for d in depths])
            self._put(self.slots, [self.kept + i for i in range(n)])
            self._put(self.masks, words)
            self._put(self.starts, [0, n])
            self._put(self.prefix, [self.kept])
            at = self.x
            for layer, (w, (write, attend)) in enumerate(zip(self.weights, self._step_descs(n))):
                self._matvec(stream, w, "qkv", self.qkv, at, n, rmsnorm=layer > 0)
                k.cache_write(write, stream=stream)
                k.attention_tree(attend, stream=stream)
                self._matvec(stream, w, "o", self.o, self.att, n)
                self._matvec(stream, w, "gate_up", self.a, self.o, n, pair_scale=1.0 / math.sqrt(cfg.ffn))
                self._matvec(stream, w, "down", self.xd, self.a, n)
                at = self.xd
            self._matvec(stream, {"head": self.head}, "head", self.logits, at, n, rmsnorm=True)
        self.parents = tuple(parents)
        return self.logits[:n]

    def _matvec(self, stream, weights, name: str, y, x, batch: int, rmsnorm: bool = False,
                pair_scale: float | None = None):
        kb, s = self.kb, self.shards[name]
        self.k.matvec(s.qtype, y, weights[name], x, s.rows, s.k, batch,
                      prologue=kb.PROLOGUE_RMSNORM if rmsnorm else kb.PROLOGUE_NONE, eps=self.cfg.eps,
                      epilogue=kb.EPILOGUE_NONE if pair_scale is None else kb.EPILOGUE_PAIR_PRODUCT,
                      pair_scale=1.0 if pair_scale is None else pair_scale, flags=kb.FLAG_WEIGHTS_STATIC,
                      stream=stream)

    def keep(self, path) -> None:
        """The last step's drafts ``path`` (from one that continues the context on, each the child of the one
        before) become the context's end."""
        path, at = list(path), -1
        for i in path:
            if not 0 <= i < len(self.parents) or self.parents[i] != at:
                raise ValueError("path must go down the last step's tree, from a draft that continues the context")
            at = i
        moves = [(self.kept + i, self.kept + j) for j, i in enumerate(path) if i != j]
        if moves:
            with self._ordered() as stream:
                self._put(self.src, [a for a, _ in moves])
                self._put(self.dst, [b for _, b in moves])
                self._put(self.starts, [0, len(moves)])
                for c in self.caches:
                    self.k.cache_move(self.kb.cache_move_desc(c, self.src, self.dst, self.starts, 1, len(moves)),
                                      stream=stream)
        self.kept += len(path)
        self.parents = ()
