"""AdamW over all tensors of a network in one launch (the reference's UpdateAdamOptimizer,
Prod/GPU/Kernels/SinglePrecision.cu:19, one launch per tensor, with decoupled weight decay) on GPUTensor."""
import ctypes

from .gpu_tensor import GPUTensor, pointer_on
from .hiplib import AdamwStepDesc, AdamwTensor, TYPES, check_status


class AdamW:
    """The optimizer: the moments of every tensor and the library's plan over them.

    parameters are float32, gradients float32 or bfloat16; copies (optional, bfloat16, None for a tensor without one) receive
    the new parameters for the bf16-stored products.  weightDecay is one value or one per tensor.  stateBits = 8 keeps the
    moments in 8 bits and a byte per 256 elements (include/sharpnet_hip.h, snhip_adamw_create), rounded at random from
    ``seed``.  states: per tensor [m, v] (float32) or [m, v, mScale, vScale] (uint8) to go on with, else zeros.  step: steps
    that have been taken."""

    def __init__(self, parameters, gradients, learningRate=1e-3, beta1=0.9, beta2=0.999, epsilon=1e-8, weightDecay=0.01, stateBits=32,
                 seed=0, states=None, copies=None, step=0):
        count = len(parameters)
        decay = list(weightDecay) if isinstance(weightDecay, (list, tuple)) else [weightDecay] * count
        copies = copies if copies is not None else [None] * count
        if len(gradients) != count or len(decay) != count or len(copies) != count or (states is not None and len(states) != count):
            raise ValueError("%d parameters need as many gradients, weight decays, states and copies" % count)
        if stateBits not in (8, 32):
            raise ValueError("stateBits is 8 or 32, not %r" % (stateBits,))
        self.LearningRate, self.Beta1, self.Beta2, self.Epsilon = learningRate, beta1, beta2, epsilon
        self.StateBits, self.Seed, self.StepCount = stateBits, int(seed), int(step)
        self._plan, self._disposed = None, False
        for p, g, c in zip(parameters, gradients, copies):
            if p.Type != "float32" or g.Type not in ("float32", "bfloat16") or (c is not None and c.Type != "bfloat16"):
                raise ValueError("parameters are float32, gradients float32 or bfloat16, copies bfloat16")
            if g.Count != p.Count or (c is not None and c.Count != p.Count):
                raise ValueError("a gradient or copy of %s does not fit its parameters of %s" % (g.Shape, p.Shape))
        if states is None:
            states = [self._zero_states(p, parameters[0].Wrapper) for p in parameters]
            if count:
                parameters[0].Wrapper.synchronize()  # (the steps may go to another stream)
        for p, s in zip(parameters, states):
            self._check_states(p, s)
        # the plan holds addresses: everything it points at stays alive with it
        self.Parameters, self.Gradients, self.States, self.Copies = list(parameters), list(gradients), [list(s) for s in states], list(copies)
        memory = (t._owner or t for tensors in zip(self.Parameters, self.Gradients, self.Copies, *zip(*self.States)) for t in tensors if t is not None)
        self._memory = list({id(t): t for t in memory}.values())
        if not count:
            return
        self._lib, self._wrapper = parameters[0]._lib, parameters[0].Wrapper
        w = self._wrapper
        table = (AdamwTensor * count)()
        for e, p, g, s, c, d in zip(table, parameters, gradients, self.States, copies, decay):
            e.parameter, e.gradient = pointer_on(w, p), pointer_on(w, g)
            e.moment1, e.moment2 = pointer_on(w, s[0]), pointer_on(w, s[1])
            if stateBits == 8:
                e.scale1, e.scale2 = pointer_on(w, s[2]), pointer_on(w, s[3])
            e.bf16_copy = pointer_on(w, c)
            e.count, e.gradient_type, e.weight_decay = p.Count, TYPES[g.Type], d
        plan = ctypes.c_void_p()
        check_status(self._lib.snhip_adamw_create(self._wrapper.handle, table, count, stateBits, ctypes.byref(plan)), "snhip_adamw_create")
        self._plan = plan

    def _zero_states(self, p, wrapper):
        if self.StateBits == 32:
            made = [GPUTensor(p.Shape, None, wrapper) for _ in range(2)]
        else:
            made = [GPUTensor([n], None, wrapper, element_type="uint8") for n in (p.Count, p.Count, -(-p.Count // 256), -(-p.Count // 256))]
        for t in made:
            t.ZeroMemory()
        return made

    def _check_states(self, p, s):
        if self.StateBits == 32:
            ok = len(s) == 2 and all(t.Type == "float32" and t.Count == p.Count for t in s)
        else:
            ok = len(s) == 4 and all(t.Type == "uint8" for t in s) and s[0].Count == s[1].Count == p.Count and \
                s[2].Count == s[3].Count == -(-p.Count // 256)
        if not ok:
            raise ValueError("the states of a tensor of %s do not fit %d-bit moments" % (p.Shape, self.StateBits))

    def Step(self, learningRate=None, gradientScale=1.0):
        """One step with the gradients as they are, times gradientScale (1 / loss scale, or a clipping factor)."""
        if self._disposed:
            raise RuntimeError("AdamW is disposed")
        for t in self._memory:
            if t._disposed:
                raise RuntimeError("memory of the optimizer's tensors is disposed")
        if learningRate is not None:
            self.LearningRate = learningRate
        if self._plan is not None:
            step = self.StepCount + 1
            if step > 0x7FFFFFFF:
                raise ValueError("step %d" % step)
            d = AdamwStepDesc()
            d.step, d.learning_rate, d.beta1, d.beta2 = step, self.LearningRate, self.Beta1, self.Beta2
            d.epsilon, d.gradient_scale, d.seed = self.Epsilon, gradientScale, self.Seed
            check_status(self._lib.snhip_adamw_step(self._wrapper.handle, self._plan, ctypes.byref(d)), "snhip_adamw_step")
        self.StepCount += 1

    def Dispose(self):
        """Ends the plan (and with it a captured graph's steps); tensors stay with whoever holds them."""
        self._disposed = True
        plan, self._plan = self._plan, None
        if plan is not None:
            self._wrapper.synchronize()
            check_status(self._lib.snhip_adamw_destroy(plan), "snhip_adamw_destroy")

    def __del__(self):
        try:
            self.Dispose()
        except Exception:
            pass
