"""Thin PyTorch custom ops (`torch.ops.marl_amd.*`) over the C ABI of libmarl_env.so.

Each op launches one HIP kernel on torch's current stream and returns / mutates device
tensors; fake (meta) implementations are registered so the ops trace under torch.compile.
The stage ops mirror the reference's pure functions:

    adjacency_bits      physics/communication_graph.py:41-105   compute_adjacency_matrix
    jam_mask_bits       physics/jamming.py:151-247              compute_disrupted_links
    lambda2_from_bits   physics/communication_graph.py:184-286  compute_laplacian + compute_lambda2
    dbscan_labels       clustering/dbscan_clustering.py:78-144  DBSCANClusterer.fit
    gae                 agents/rollout_buffer.py:151-204        compute_returns_and_advantages
    reward_per_agent    environment/reward.py:308-396           RewardCalculator.compute_per_agent
    reward_obs          environment/reward.py:106-176, observation.py:264-332   compute + build_vectorized
    env_step            environment/jammer_env.py:356-457       JammerEnv.step (state mutated in place)

The operators of a residual policy trunk and of the draw from its head have no counterpart in the reference; the first
three are differentiable (the dropout twice, the others once), all take float32, bfloat16 and float16:

    gated_linear(x, w_gate, w_up, act)                              act(x w_gate^T) * (x w_up^T)
    residual_norm(x, block, w_post, w_pre, gate, scale, eps, kind)  y = scale x + gate N(block; w_post), n = N(y; w_pre)
    keyed_dropout(x, p, seed, keys)                                 mask from (seed, row key, column), never stored
    sample_logits(logits, u, temperature, top_k, top_p, min_p)      index and log-probability of a filtered draw

Bit matrices are int32 tensors [E, N, ceil(N/32)]: row i, bit j of word j // 32.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import List, Optional, Tuple

import torch

from . import _lib
from .env import BatchedJammerEnv, EnvConfig


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


@lru_cache(maxsize=64)
def _params(N: int, M: int, P_tx_dbm: float, P_sens_dbm: float, P_jammer_dbm: float, P_jam_thresh_dbm: float,
            eps: float, min_samples: int, arena_size: float):
    return EnvConfig(N=N, M=M, P_tx_dbm=P_tx_dbm, P_sens_dbm=P_sens_dbm, P_jammer_dbm=P_jammer_dbm,
                     P_jam_thresh_dbm=P_jam_thresh_dbm, eps=eps, min_samples=min_samples,
                     arena_size=arena_size).to_params()


def _check_dev(*ts):
    for t in ts:
        if t is not None and (not t.is_cuda or not t.is_contiguous()):
            raise ValueError("marl_amd ops need contiguous tensors on the HIP device")


@torch.library.custom_op("marl_amd::adjacency_bits", mutates_args=())
def adjacency_bits(x: torch.Tensor, y: torch.Tensor, band: torch.Tensor, P_tx_dbm: float = 20.0,
                   P_sens_dbm: float = -90.0) -> torch.Tensor:
    """x, y [E,N] float64, band [E] int32 -> adjacency bits."""
    _check_dev(x, y, band)
    E, N = x.shape
    p = _params(N, 1, P_tx_dbm, P_sens_dbm, 30.0, -70.0, 30.0, 2, 200.0)
    out = torch.zeros(E, N, (N + 31) // 32, dtype=torch.int32, device=x.device)
    _lib.check(_lib.load().marl_adjacency_bits(C.byref(p), E, x.data_ptr(), y.data_ptr(), band.data_ptr(),
                                               out.data_ptr(), _stream()), "marl_adjacency_bits")
    return out


@adjacency_bits.register_fake
def _(x, y, band, P_tx_dbm=20.0, P_sens_dbm=-90.0):
    E, N = x.shape
    return x.new_empty((E, N, (N + 31) // 32), dtype=torch.int32)


@torch.library.custom_op("marl_amd::jam_mask_bits", mutates_args=())
def jam_mask_bits(x: torch.Tensor, y: torch.Tensor, band: torch.Tensor, jam_x: torch.Tensor, jam_y: torch.Tensor,
                  jam_band: torch.Tensor, P_jammer_dbm: float = 30.0, P_jam_thresh_dbm: float = -70.0) -> torch.Tensor:
    """Enemy x, y [E,N], band [E]; jammer jam_x, jam_y [E,M] float64, jam_band [E,M] int32 -> mask bits."""
    _check_dev(x, y, band, jam_x, jam_y, jam_band)
    E, N = x.shape
    M = jam_x.shape[1]
    p = _params(N, M, 20.0, -90.0, P_jammer_dbm, P_jam_thresh_dbm, 30.0, 2, 200.0)
    out = torch.zeros(E, N, (N + 31) // 32, dtype=torch.int32, device=x.device)
    _lib.check(_lib.load().marl_jam_mask_bits(C.byref(p), E, x.data_ptr(), y.data_ptr(), band.data_ptr(),
                                              jam_x.data_ptr(), jam_y.data_ptr(), jam_band.data_ptr(),
                                              out.data_ptr(), _stream()), "marl_jam_mask_bits")
    return out


@jam_mask_bits.register_fake
def _(x, y, band, jam_x, jam_y, jam_band, P_jammer_dbm=30.0, P_jam_thresh_dbm=-70.0):
    E, N = x.shape
    return x.new_empty((E, N, (N + 31) // 32), dtype=torch.int32)


@torch.library.custom_op("marl_amd::lambda2_from_bits", mutates_args=())
def lambda2_from_bits(bits: torch.Tensor, rounds: int = 0) -> torch.Tensor:
    """bits [E,N,W] int32 -> lambda2 [E] float64."""
    _check_dev(bits)
    E, N, _ = bits.shape
    lib = _lib.load()
    out = torch.zeros(E, dtype=torch.float64, device=bits.device)
    nb = lib.marl_lambda2_workspace_bytes(N, E)
    ws = torch.empty(nb, dtype=torch.uint8, device=bits.device) if nb else None
    _lib.check(lib.marl_lambda2_from_bits(N, E, bits.data_ptr(), out.data_ptr(), rounds,
                                          ws.data_ptr() if ws is not None else None, _stream()),
               "marl_lambda2_from_bits")
    return out


@lambda2_from_bits.register_fake
def _(bits, rounds=0):
    return bits.new_empty((bits.shape[0],), dtype=torch.float64)


@torch.library.custom_op("marl_amd::dbscan_labels", mutates_args=())
def dbscan_labels(x: torch.Tensor, y: torch.Tensor, eps: float, min_samples: int = 2,
                  arena_size: float = 200.0) -> List[torch.Tensor]:
    """x, y [E,N] float64 -> [labels [E,N] i32, cent_x [E,N+1] f64, cent_y, cent_size i32, n_clusters [E], ncent [E]]."""
    _check_dev(x, y)
    E, N = x.shape
    p = _params(N, 1, 20.0, -90.0, 30.0, -70.0, eps, min_samples, arena_size)
    dev = x.device
    labels = torch.zeros(E, N, dtype=torch.int32, device=dev)
    cx = torch.zeros(E, N + 1, dtype=torch.float64, device=dev)
    cy = torch.zeros(E, N + 1, dtype=torch.float64, device=dev)
    csz = torch.zeros(E, N + 1, dtype=torch.int32, device=dev)
    ncl = torch.zeros(E, dtype=torch.int32, device=dev)
    nce = torch.zeros(E, dtype=torch.int32, device=dev)
    _lib.check(_lib.load().marl_dbscan(C.byref(p), E, x.data_ptr(), y.data_ptr(), labels.data_ptr(), cx.data_ptr(),
                                       cy.data_ptr(), csz.data_ptr(), ncl.data_ptr(), nce.data_ptr(), _stream()),
               "marl_dbscan")
    return [labels, cx, cy, csz, ncl, nce]


@dbscan_labels.register_fake
def _(x, y, eps, min_samples=2, arena_size=200.0):
    E, N = x.shape
    i32, f64 = torch.int32, torch.float64
    return [x.new_empty((E, N), dtype=i32), x.new_empty((E, N + 1), dtype=f64), x.new_empty((E, N + 1), dtype=f64),
            x.new_empty((E, N + 1), dtype=i32), x.new_empty((E,), dtype=i32), x.new_empty((E,), dtype=i32)]


@torch.library.custom_op("marl_amd::gae", mutates_args=())
def gae(rewards: torch.Tensor, values: torch.Tensor, dones: torch.Tensor, last_value: torch.Tensor,
        last_done: torch.Tensor, gamma: float = 0.99, lam: float = 0.95) -> List[torch.Tensor]:
    """rewards, values, dones [T,E] float32; last_value, last_done [E] -> [advantages, returns] [T,E]."""
    _check_dev(rewards, values, dones, last_value, last_done)
    T, E = rewards.shape
    adv, ret = torch.zeros_like(rewards), torch.zeros_like(rewards)
    _lib.check(_lib.load().marl_gae(T, E, rewards.data_ptr(), values.data_ptr(), dones.data_ptr(),
                                    last_value.data_ptr(), last_done.data_ptr(), gamma, lam, adv.data_ptr(),
                                    ret.data_ptr(), _stream()), "marl_gae")
    return [adv, ret]


@gae.register_fake
def _(rewards, values, dones, last_value, last_done, gamma=0.99, lam=0.95):
    return [torch.empty_like(rewards), torch.empty_like(rewards)]


@torch.library.custom_op("marl_amd::reward_per_agent", mutates_args=())
def reward_per_agent(state: torch.Tensor, handle: int, lambda2: torch.Tensor) -> torch.Tensor:
    """Per-jammer reward [E,M] float32 of the registered env's current state for the given lambda2 [E] f64."""
    env = _ENVS[handle]
    if state.data_ptr() != env._buf.data_ptr():
        raise ValueError("state must be the buffer of the registered env")
    _check_dev(lambda2)
    return env.reward_per_agent(lambda2)


@reward_per_agent.register_fake
def _(state, handle, lambda2):
    env = _ENVS[handle]
    return lambda2.new_empty((env.E, env.M), dtype=torch.float32)


@torch.library.custom_op("marl_amd::reward_obs", mutates_args=())
def reward_obs(state: torch.Tensor, handle: int, lambda2: torch.Tensor) -> List[torch.Tensor]:
    """Reward stage + observation stage of the registered env's current state for the given lambda2 [E] f64:
    [reward [E] f32, reward_terms [E,5] f32, obs [E,M,5] f32, avg_jamming_power_dbm [E] f64]."""
    env = _ENVS[handle]
    if state.data_ptr() != env._buf.data_ptr():
        raise ValueError("state must be the buffer of the registered env")
    _check_dev(lambda2)
    v, dev = env.views, env.device
    io = _lib.MarlRewardObsIO()
    rew = torch.empty(env.E, dtype=torch.float32, device=dev)
    terms = torch.empty(env.E, 5, dtype=torch.float32, device=dev)
    obs = torch.empty(env.E, env.M, 5, dtype=torch.float32, device=dev)
    avgp = torch.empty(env.E, dtype=torch.float64, device=dev)
    io.lambda2, io.lambda2_initial = lambda2.data_ptr(), v["lambda2_initial"].data_ptr()
    for name in ("enemy_band", "enemy_x", "enemy_y", "jam_x", "jam_y", "jam_band", "cent_x", "cent_y", "cent_size",
                 "n_clusters", "ncent", "assign"):
        setattr(io, name, v[name].data_ptr())
    io.vx, io.vy = v["last_vx"].data_ptr(), v["last_vy"].data_ptr()
    io.reward, io.reward_terms, io.obs, io.avg_power_dbm = rew.data_ptr(), terms.data_ptr(), obs.data_ptr(), avgp.data_ptr()
    _lib.check(_lib.load().marl_reward_obs(C.byref(env.params), env.E, C.byref(io), _stream()), "marl_reward_obs")
    return [rew, terms, obs, avgp]


@reward_obs.register_fake
def _(state, handle, lambda2):
    env = _ENVS[handle]
    f32 = torch.float32
    return [lambda2.new_empty((env.E,), dtype=f32), lambda2.new_empty((env.E, 5), dtype=f32),
            lambda2.new_empty((env.E, env.M, 5), dtype=f32), lambda2.new_empty((env.E,), dtype=torch.float64)]


# -- the step itself: state lives in a BatchedJammerEnv, addressed by a small integer handle -------
_ENVS = {}


def register_env(env: BatchedJammerEnv) -> int:
    h = len(_ENVS) + 1
    _ENVS[h] = env
    return h


@torch.library.custom_op("marl_amd::env_step", mutates_args=("state", "obs", "reward", "truncated"))
def env_step(state: torch.Tensor, handle: int, actions: torch.Tensor, noise: Optional[torch.Tensor],
             obs: torch.Tensor, reward: torch.Tensor, truncated: torch.Tensor) -> None:
    """JammerEnv.step for every env of the registered batch: `state` is its device state buffer
    (mutated), obs [E,M,5] f32 / reward [E] f32 / truncated [E] u8 receive the results."""
    env = _ENVS[handle]
    if state.data_ptr() != env._buf.data_ptr():
        raise ValueError("state must be the buffer of the registered env")
    auto = env.auto_reset
    env.auto_reset = False
    try:
        env.step(actions, noise, out_obs=obs, out_reward=reward, out_truncated=truncated)
    finally:
        env.auto_reset = auto


@env_step.register_fake
def _(state, handle, actions, noise, obs, reward, truncated):
    return None


# -- operators of a residual policy trunk and of the draw from its head ------------------------------------------------
# Registered on the dispatcher directly (torch.library.Library): a custom_op wrapper costs 10 us a call more, which is
# what the smallest of these calls take on the GPU.  The *_saved / *_backward forms are what autograd calls.
_LIB = torch.library.Library("marl_amd", "FRAGMENT")
_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _define(name, schema, impl, fake, autograd=None):
    _LIB.define(name + schema)
    _LIB.impl(name, impl, "CUDA")
    _LIB.impl(name, impl, "CPU")                 # the checks of the arguments, then the refusal of the device
    _LIB.impl(name, fake, "Meta")
    if autograd is not None:
        _LIB.impl(name, autograd, "AutogradCUDA")


def _need(ok, text):
    if not ok:
        raise ValueError(text)


def _same(name, *ts):
    """One supported element type and one HIP device for all of `ts` (None is skipped)."""
    first = ts[0]
    _need(first.dtype in _DTYPES, f"{name}: float32, bfloat16 or float16 tensors, not {first.dtype}")
    for t in ts[1:]:
        _need(t is None or t.dtype == first.dtype, f"{name}: all of these tensors must be {first.dtype}")
    _on_device(name, *ts)


def _on_device(name, first, *rest):
    for t in rest:
        _need(t is None or t.device == first.device, f"{name}: tensors on different devices")
    _need(first.is_cuda, f"{name}: tensors must be on the HIP device")


def _rows(t):
    """t [..., d] as (tensor, rows, row stride): without a copy if the leading dimensions are evenly spaced and the elements
    of a row adjacent, as in a slice of columns or of one dimension."""
    d = t.shape[-1]
    rows = t.numel() // d if d else 0
    if t.dim() == 2:
        if t.stride(1) == 1 and (rows == 1 or t.stride(0) >= d):
            return t, rows, max(t.stride(0), d)
    elif t.is_contiguous():
        return t, rows, d
    return t.contiguous(), rows, d


class _on:
    """Makes t's device the current one for the launches inside; gives its current stream."""

    def __init__(self, t):
        self.index, self.guard = t.device.index, None

    def __enter__(self):
        if torch.cuda.current_device() != self.index:
            self.guard = torch.cuda.device(self.index)
            self.guard.__enter__()
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _check_gated(x, w_gate, w_up, act):
    _need(act in _lib.ACTS, f"gated_linear: act must be one of {sorted(_lib.ACTS)}, not {act!r}")
    _need(w_gate.dim() == 2 and w_up.shape == w_gate.shape, "gated_linear: w_gate and w_up must be [h, d] of one shape")
    _need(x.dim() >= 1 and x.shape[-1] == w_gate.shape[1], "gated_linear: x must be [..., d] for weights [h, d]")
    _need(w_gate.shape[0] > 0 and w_gate.shape[1] > 0, "gated_linear: weights without elements")


def _gated_launch(x, w_gate, w_up, act, save):
    _check_gated(x, w_gate, w_up, act)
    _same("gated_linear", x, w_gate, w_up)
    h, d = w_gate.shape
    y = torch.empty(x.shape[:-1] + (h,), dtype=x.dtype, device=x.device)
    a, b = (torch.empty_like(y), torch.empty_like(y)) if save else (None, None)
    if y.numel():
        x, rows, ldx = _rows(x)
        w_gate, _, ldg = _rows(w_gate)
        w_up, _, ldu = _rows(w_up)
        with _on(x) as stream:
            rc = _lib.load().marl_gated_forward(_DTYPES[x.dtype], _lib.ACTS[act], rows, d, h, x.data_ptr(), ldx, w_gate.data_ptr(), ldg,
                                                w_up.data_ptr(), ldu, y.data_ptr(), a.data_ptr() if save else None,
                                                b.data_ptr() if save else None, stream)
            _lib.check(rc, "marl_gated_forward")
    return (y, a, b) if save else y


def _gated_linear(x, w_gate, w_up, act="silu"):
    return _gated_launch(x, w_gate, w_up, act, False)


def _gated_linear_saved(x, w_gate, w_up, act):
    return _gated_launch(x, w_gate, w_up, act, True)


def _gated_linear_backward(gy, x, w_gate, w_up, a, b, act, need_x, need_w):
    h, d = w_gate.shape
    dx = torch.empty(x.shape if need_x else (0,), dtype=x.dtype, device=x.device)
    dwg, dwu = (torch.empty((h, d) if need_w else (0,), dtype=x.dtype, device=x.device) for _ in range(2))
    if not x.numel():
        return dx, dwg.zero_(), dwu.zero_()
    x, rows, ldx = _rows(x)
    w_gate, _, ldg = _rows(w_gate)
    w_up, _, ldu = _rows(w_up)
    gy, _, ldgy = _rows(gy)
    lib, dt = _lib.load(), _DTYPES[x.dtype]
    with _on(x) as stream:
        ws = torch.empty(lib.marl_gated_workspace_bytes(dt, rows, d, h), dtype=torch.uint8, device=x.device)
        _lib.check(lib.marl_gated_backward(dt, _lib.ACTS[act], rows, d, h, x.data_ptr(), ldx, w_gate.data_ptr(), ldg, w_up.data_ptr(), ldu,
                                           a.data_ptr(), b.data_ptr(), gy.data_ptr(), ldgy, dx.data_ptr() if need_x else None,
                                           dwg.data_ptr() if need_w else None, dwu.data_ptr() if need_w else None, ws.data_ptr(), stream),
                   "marl_gated_backward")
    return dx, dwg, dwu


def _like(x, *shape):
    return x.new_empty(shape)


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act):
        y, a, b = torch.ops.marl_amd.gated_linear_saved(x, w_gate, w_up, act)
        ctx.save_for_backward(x, w_gate, w_up, a, b)
        ctx.act = act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        x, w_gate, w_up, a, b = ctx.saved_tensors
        nx, ng, nu, _ = ctx.needs_input_grad
        dx, dwg, dwu = torch.ops.marl_amd.gated_linear_backward(gy, x, w_gate, w_up, a, b, ctx.act, nx, ng or nu)
        return dx if nx else None, dwg if ng else None, dwu if nu else None, None


def _wants_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _gated_linear_autograd(x, w_gate, w_up, act="silu"):
    return _GatedLinear.apply(x, w_gate, w_up, act) if _wants_grad(x, w_gate, w_up) else _gated_linear(x, w_gate, w_up, act)


def _gated_fake(x, w_gate, w_up, act="silu"):
    _check_gated(x, w_gate, w_up, act)
    return _like(x, *x.shape[:-1], w_gate.shape[0])


_define("gated_linear", '(Tensor x, Tensor w_gate, Tensor w_up, str act="silu") -> Tensor', _gated_linear, _gated_fake, _gated_linear_autograd)
_define("gated_linear_saved", "(Tensor x, Tensor w_gate, Tensor w_up, str act) -> (Tensor, Tensor, Tensor)", _gated_linear_saved,
        lambda x, wg, wu, act: tuple(_gated_fake(x, wg, wu, act) for _ in range(3)))
_define("gated_linear_backward", "(Tensor gy, Tensor x, Tensor w_gate, Tensor w_up, Tensor a, Tensor b, str act, bool need_x, bool need_w)"
        " -> (Tensor, Tensor, Tensor)", _gated_linear_backward,
        lambda gy, x, wg, wu, a, b, act, nx, nw: (_like(x, *(x.shape if nx else (0,))), *(_like(x, *(wg.shape if nw else (0,))) for _ in range(2))))


def _check_norm(x, block, w_post, w_pre, gate, eps, kind):
    _need(kind in _lib.NORMS, f"residual_norm: kind must be one of {sorted(_lib.NORMS)}, not {kind!r}")
    _need(x.dim() >= 1 and block.shape == x.shape, "residual_norm: x and block must be [..., d] of one shape")
    d = x.shape[-1]
    _need(0 < d <= _lib.MAX_NORM_WIDTH, f"residual_norm: rows of 1 to {_lib.MAX_NORM_WIDTH} elements, not {d}")
    _need(w_post.shape == (d,) and w_pre.shape == (d,), "residual_norm: w_post and w_pre must be [d]")
    _need(gate is None or gate.shape == (d,) or gate.shape == x.shape, "residual_norm: gate must be [d] or shaped like x")
    _need(eps >= 0.0, "residual_norm: eps must not be negative")


def _gate_rows(gate, x):
    """Pointer and row stride of the gate: stride 0 for one gate for all rows."""
    if gate is None:
        return None, None, 0
    if gate.dim() == 1 and x.dim() > 1:
        gate = gate.contiguous()
        return gate, gate.data_ptr(), 0
    gate, _, ld = _rows(gate)
    return gate, gate.data_ptr(), ld


def _norm_launch(x, block, w_post, w_pre, gate, scale, eps, kind, save):
    _check_norm(x, block, w_post, w_pre, gate, eps, kind)
    _same("residual_norm", x, block, w_post, w_pre, gate)
    y, n = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for _ in range(2))
    stats = torch.empty(x.shape[:-1] + (4,), dtype=torch.float32, device=x.device) if save else None
    if x.numel():
        d = x.shape[-1]
        gate, pg, ldg = _gate_rows(gate, x)
        x, rows, ldx = _rows(x)
        block, _, ldb = _rows(block)
        w_post, w_pre = w_post.contiguous(), w_pre.contiguous()
        with _on(x) as stream:
            _lib.check(_lib.load().marl_residual_norm(_DTYPES[x.dtype], _lib.NORMS[kind], rows, d, x.data_ptr(), ldx, block.data_ptr(), ldb,
                                                      w_post.data_ptr(), w_pre.data_ptr(), pg, ldg, scale, eps, y.data_ptr(), n.data_ptr(),
                                                      stats.data_ptr() if save else None, stream), "marl_residual_norm")
    return (y, n, stats) if save else (y, n)


def _residual_norm(x, block, w_post, w_pre, gate=None, scale=1.0, eps=1e-5, kind="rms"):
    return _norm_launch(x, block, w_post, w_pre, gate, scale, eps, kind, False)


def _residual_norm_saved(x, block, w_post, w_pre, gate, scale, eps, kind):
    return _norm_launch(x, block, w_post, w_pre, gate, scale, eps, kind, True)


def _residual_norm_backward(gy, gn, y, block, w_post, w_pre, gate, stats, scale, kind):
    dx, db = (torch.empty(y.shape, dtype=y.dtype, device=y.device) for _ in range(2))
    d = y.shape[-1]
    dpost, dpre = (torch.empty(d, dtype=y.dtype, device=y.device) for _ in range(2))
    dgate = torch.empty(gate.shape if gate is not None else (0,), dtype=y.dtype, device=y.device)
    if not y.numel():
        return dx, db, dpost.zero_(), dpre.zero_(), dgate.zero_()
    gate, pg, ldg = _gate_rows(gate, y)
    block, rows, ldb = _rows(block)
    w_post, w_pre = w_post.contiguous(), w_pre.contiguous()
    gy, ldgy = (None, 0) if gy is None else _rows(gy)[::2]
    gn, ldgn = (None, 0) if gn is None else _rows(gn)[::2]
    lib = _lib.load()
    with _on(y) as stream:
        ws = torch.empty(lib.marl_residual_norm_workspace_bytes(d), dtype=torch.uint8, device=y.device)
        _lib.check(lib.marl_residual_norm_backward(
            _DTYPES[y.dtype], _lib.NORMS[kind], rows, d, y.data_ptr(), block.data_ptr(), ldb, w_post.data_ptr(), w_pre.data_ptr(), pg, ldg,
            stats.data_ptr(), None if gy is None else gy.data_ptr(), ldgy, None if gn is None else gn.data_ptr(), ldgn, scale, dx.data_ptr(),
            db.data_ptr(), dpost.data_ptr(), dpre.data_ptr(), dgate.data_ptr() if pg is not None else None, ws.data_ptr(), stream),
            "marl_residual_norm_backward")
    return dx, db, dpost, dpre, dgate


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, block, w_post, w_pre, gate, scale, eps, kind):
        y, n, stats = torch.ops.marl_amd.residual_norm_saved(x, block, w_post, w_pre, gate, scale, eps, kind)
        ctx.save_for_backward(y, block, w_post, w_pre, gate, stats)
        ctx.scale, ctx.kind = scale, kind
        ctx.set_materialize_grads(False)
        return y, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, gn):
        y, block, w_post, w_pre, gate, stats = ctx.saved_tensors
        if gy is None and gn is None:
            return (None,) * 8
        out = torch.ops.marl_amd.residual_norm_backward(gy, gn, y, block, w_post, w_pre, gate, stats, ctx.scale, ctx.kind)
        need = ctx.needs_input_grad
        return tuple(g if need[i] else None for i, g in enumerate(out)) + (None,) * 3


def _residual_norm_autograd(x, block, w_post, w_pre, gate=None, scale=1.0, eps=1e-5, kind="rms"):
    f = _ResidualNorm.apply if _wants_grad(x, block, w_post, w_pre, gate) else _residual_norm
    return f(x, block, w_post, w_pre, gate, scale, eps, kind)


def _norm_fake(x, block, w_post, w_pre, gate=None, scale=1.0, eps=1e-5, kind="rms"):
    _check_norm(x, block, w_post, w_pre, gate, eps, kind)
    return _like(x, *x.shape), _like(x, *x.shape)


_define("residual_norm", '(Tensor x, Tensor block, Tensor w_post, Tensor w_pre, Tensor? gate=None, float scale=1.0, float eps=1e-5, '
        'str kind="rms") -> (Tensor, Tensor)', _residual_norm, _norm_fake, _residual_norm_autograd)
_define("residual_norm_saved", "(Tensor x, Tensor block, Tensor w_post, Tensor w_pre, Tensor? gate, float scale, float eps, str kind)"
        " -> (Tensor, Tensor, Tensor)", _residual_norm_saved,
        lambda x, *r: _norm_fake(x, *r) + (x.new_empty((*x.shape[:-1], 4), dtype=torch.float32),))
_define("residual_norm_backward", "(Tensor? gy, Tensor? gn, Tensor y, Tensor block, Tensor w_post, Tensor w_pre, Tensor? gate, Tensor stats, "
        "float scale, str kind) -> (Tensor, Tensor, Tensor, Tensor, Tensor)", _residual_norm_backward,
        lambda gy, gn, y, block, wo, wr, gate, st, s, k: (_like(y, *y.shape), _like(y, *y.shape), _like(y, y.shape[-1]), _like(y, y.shape[-1]),
                                                          _like(y, *(gate.shape if gate is not None else (0,)))))


def _check_dropout(x, p, keys):
    _need(x.dim() >= 1 and 0.0 <= p <= 1.0, "keyed_dropout: x must be [..., d] and p in [0, 1]")
    _need(keys is None or (keys.dtype == torch.int64 and keys.shape == x.shape[:-1]), "keyed_dropout: keys must be int64, one per row of x")


def _dropout_impl(x, p, seed, keys=None):
    _check_dropout(x, p, keys)
    _same("keyed_dropout", x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if keys is not None:
        _on_device("keyed_dropout", x, keys)
        keys = keys.contiguous()
    if x.numel():
        x, rows, ldx = _rows(x)
        with _on(x) as stream:
            _lib.check(_lib.load().marl_keyed_dropout(_DTYPES[x.dtype], rows, x.shape[-1], x.data_ptr(), ldx, y.data_ptr(),
                                                      None if keys is None else keys.data_ptr(), p, seed & 0xFFFFFFFFFFFFFFFF, stream),
                       "marl_keyed_dropout")
    return y


class _KeyedDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, keys):
        ctx.save_for_backward(keys)
        ctx.p, ctx.seed = p, seed
        return torch.ops.marl_amd.keyed_dropout(x.detach(), p, seed, keys)

    @staticmethod
    def backward(ctx, gy):                        # linear in x: differentiable again through the same op
        return torch.ops.marl_amd.keyed_dropout(gy, ctx.p, ctx.seed, ctx.saved_tensors[0]), None, None, None


def _dropout_autograd(x, p, seed, keys=None):
    return (_KeyedDropout.apply if _wants_grad(x) else _dropout_impl)(x, p, seed, keys)


def _dropout_fake(x, p, seed, keys=None):
    _check_dropout(x, p, keys)
    return _like(x, *x.shape)


_define("keyed_dropout", "(Tensor x, float p, int seed, Tensor? keys=None) -> Tensor", _dropout_impl, _dropout_fake, _dropout_autograd)


def _check_sample(logits, u, temperature, top_k, top_p, min_p, settings):
    V = logits.shape[-1] if logits.dim() else 0
    _need(0 < V <= _lib.MAX_CHOICES, f"sample_logits: logits must be [..., V] with V from 1 to {_lib.MAX_CHOICES}")
    _need(u.shape == logits.shape[:-1] and u.dtype == torch.float32, "sample_logits: u must be float32, one number per row")
    if settings is None:
        _need(temperature >= 0.0 and top_k >= 0 and top_p > 0.0 and 0.0 <= min_p <= 1.0,
              "sample_logits: temperature >= 0, top_k >= 0, top_p > 0 and min_p in [0, 1]")
    else:
        _need(settings.shape == (*logits.shape[:-1], 4) and settings.dtype == torch.float32,
              "sample_logits: settings must be float32 [..., 4]: temperature, top_k, top_p, min_p of every row")


def _sample_impl(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, *, settings=None):
    _check_sample(logits, u, temperature, top_k, top_p, min_p, settings)
    _same("sample_logits", logits)
    _on_device("sample_logits", logits, u, settings)
    V = logits.shape[-1]
    index = torch.empty(u.shape, dtype=torch.int64, device=u.device)
    log_prob = torch.empty(u.shape, dtype=torch.float32, device=u.device)
    if u.numel():
        logits, rows, ld = _rows(logits)
        u = u.contiguous()
        settings = None if settings is None else settings.contiguous()
        with _on(logits) as stream:
            _lib.check(_lib.load().marl_sample_logits(_DTYPES[logits.dtype], rows, V, logits.data_ptr(), ld, u.data_ptr(), temperature,
                                                      min(top_k, _lib.MAX_CHOICES), top_p, min_p, None if settings is None else settings.data_ptr(),
                                                      index.data_ptr(), log_prob.data_ptr(), stream), "marl_sample_logits")
    return index, log_prob


def _sample_fake(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, *, settings=None):
    _check_sample(logits, u, temperature, top_k, top_p, min_p, settings)
    return u.new_empty(u.shape, dtype=torch.int64), u.new_empty(u.shape)


_define("sample_logits", "(Tensor logits, Tensor u, float temperature=1.0, int top_k=0, float top_p=1.0, float min_p=0.0, *, "
        "Tensor? settings=None) -> (Tensor, Tensor)", _sample_impl, _sample_fake)
